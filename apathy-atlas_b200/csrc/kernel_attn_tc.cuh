// Paged attention for many rows (chunks of a prompt, and few-token chunks with many heads to a KV head): tcgen05.
//
// A block is two tiles of 128 rows (DP 256: one), each with scores S = Q K^T [128 x 128] and an output O [128 x DP] in tensor memory:
//     S_g (128 columns each) | O_g (DP columns each)      P_g, BF16, over the first half of S_g's columns
// One thread owns a row: 128 scores come to its registers (tcgen05.ld), maximum and sum need no exchange with other threads, P goes back
// to tensor memory as the A operand of O += P V.  The two tiles take turns: while one's scores are in its softmax, the tensor cores work on
// the other's P V and next Q K^T.  Q, K, V are 128-byte-swizzled tiles in shared memory: Q and K K-major, V as it lies in the cache
// ([key][channel]), the MN-major form of the B operand.  K and V come page by page by TMA, in boxes of the largest power of two that
// divides page and tile (8 rows at least); zero fill stands in for pages that do not exist and for channels behind head_dim.
//
// O is multiplied with 2^(M_old - M_new) only where a row's maximum has grown by more than 2^8 (RESCALE) since O's last factor: until then
// the weights are 2^(s - M) with the old M, up to 2^8 and in the same FP32 sums, which is the same quotient.  That takes the
// correction off the path of nearly every tile.
//
// Warps: 0 TMA, 1 MMA (converged, one lane issues), 2 tensor memory; 4-7 and 8-11 softmax, epilogue and Q of a tile each; E4M3 caches:
// 12-15 turn raw tiles into FP16 ones (one instruction for two values, exact, NaN kept; Q as FP16 with a power of two per row, see the
// mma.sync form).  Every wait is bounded as elsewhere in the library.
#pragma once

#include "kernel_attn.cuh"
#include "kernel_tc.cuh"

namespace atlas {
namespace attn {

using namespace atlas::tc;

constexpr uint32_t TC_KEYS = 128, TC_TILE_ROWS = 128;
constexpr float TC_RESCALE = 8.0f;

template <int DP, bool FP8> struct TcCfg {
    static constexpr int NQ = DP <= 128 ? 2 : 1;                             // row tiles
    static constexpr int ROWS = NQ * int(TC_TILE_ROWS);
    static constexpr int PANELS = DP / 64;                                   // 128-byte panels of a row
    static constexpr int PANEL = 128 * 128;
    static constexpr int TILE = PANELS * PANEL;                              // Q of a row tile; K or V of a key tile
    static constexpr int STAGES = DP <= 64 ? 4 : DP <= 128 ? 2 : 1;
    static constexpr int RAW = FP8 ? 128 * DP : 0, RAW_STAGES = FP8 ? (DP <= 128 ? 2 : 1) : 0;
    static constexpr int OFF_Q = 0, OFF_K = NQ * TILE, OFF_V = OFF_K + STAGES * TILE, OFF_RAW = OFF_V + STAGES * TILE;
    static constexpr int OFF_SCALE = OFF_RAW + RAW_STAGES * RAW;             // float[ROWS]: E4M3: what takes a row's power of two back
    static constexpr int OFF_BAR = OFF_SCALE + (FP8 ? ROWS * 4 : 0);
    static constexpr int N_BAR = 4 * STAGES + 1 + 4 * NQ + 2 * RAW_STAGES;
    static constexpr int OFF_MISC = OFF_BAR + N_BAR * 8;                     // tensor memory, -, abort; attn_find's words
    static constexpr int SMEM = OFF_MISC + 16 + 20 * 8 + 1024;
    static constexpr int SOFT_WARPS = 4 * NQ, WARPS = 4 + SOFT_WARPS + (FP8 ? 4 : 0), THREADS = 32 * WARPS;
    static constexpr int CONV_WARP0 = 4 + SOFT_WARPS;
    // registers a thread: at launch, and the split (warpgroups of 4 warps; the sum of the split is at most the launch's)
    static constexpr int LAUNCH_REGS = THREADS <= 256 ? 248 : THREADS <= 384 ? 168 : 128;
    static constexpr int SOFT_REGS = THREADS <= 256 ? 248 : THREADS <= 384 ? (FP8 ? 248 : 200) : 168;
    static constexpr int AUX_REGS = THREADS <= 256 ? 248 : THREADS <= 384 ? (FP8 ? 128 : 104) : 88;
    static_assert(32 * (SOFT_WARPS * SOFT_REGS + (WARPS - SOFT_WARPS) * AUX_REGS) <= THREADS * LAUNCH_REGS, "registers");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
          "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
          "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// V as it lies in the cache: rows of keys, channels contiguous.  MN-major, 128-byte swizzle: 64 channels x 8 keys an atom of 1024 bytes,
// the next 8 keys 1024 bytes on (stride offset), the next 64 channels a panel on (leading offset).
__device__ __forceinline__ uint64_t make_mnmajor_sw128_desc(uint32_t smem_addr, uint32_t panel_bytes) {
    return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(panel_bytes >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// kind::f16, FP32 accumulator, A K-major; both operands BF16, or FP16; B K-major, or MN-major
__host__ __device__ constexpr uint32_t attn_idesc(uint32_t n, bool half, bool b_mn) {
    return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

template <bool HALF> __device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_bf16x2(a, b);
    }
}

template <int DP, bool FP8>
__global__ void __launch_bounds__(TcCfg<DP, FP8>::THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p, const uint32_t box_rows) {
    using C = TcCfg<DP, FP8>;
    constexpr int NQ = C::NQ, ST = C::STAGES;
    extern __shared__ uint8_t attn_smem_raw[];
    const uint32_t base = (smem_u32(attn_smem_raw) + 1023u) & ~1023u;
    uint8_t* const gen = attn_smem_raw + (base - smem_u32(attn_smem_raw));
    const uint32_t bar = base + C::OFF_BAR;
    const uint32_t K_FULL = bar, K_EMPTY = bar + 8 * ST, V_FULL = bar + 16 * ST, V_EMPTY = bar + 24 * ST, V_TAIL = bar + 32 * ST, Q_FULL = V_TAIL + 8,
                   S_FULL = Q_FULL + 8 * NQ, P_FULL = S_FULL + 8 * NQ, PV_DONE = P_FULL + 8 * NQ, RAW_FULL = PV_DONE + 8 * NQ, RAW_EMPTY = RAW_FULL + 8 * C::RAW_STAGES;
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(gen + C::OFF_MISC);
    volatile uint32_t* const abort_flag = misc + 2;
    uint64_t* const sh = reinterpret_cast<uint64_t*>(gen + C::OFF_MISC + 16);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(K_FULL + 8 * i, FP8 ? 128 : 1); mbar_init(K_EMPTY + 8 * i, 1); mbar_init(V_FULL + 8 * i, FP8 ? 128 : 1); mbar_init(V_EMPTY + 8 * i, 1);
        }
        mbar_init(V_TAIL, 1);
        for (int g = 0; g < NQ; ++g) { mbar_init(Q_FULL + 8 * g, 128); mbar_init(S_FULL + 8 * g, 1); mbar_init(P_FULL + 8 * g, 128); mbar_init(PV_DONE + 8 * g, 1); }
        for (int i = 0; i < C::RAW_STAGES; ++i) { mbar_init(RAW_FULL + 8 * i, 1); mbar_init(RAW_EMPTY + 8 * i, 128); }
        misc[2] = 0;
        fence_barrier_init();
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    if (warp == 2) { tmem_alloc(base + C::OFF_MISC, 512); tmem_relinquish(); }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = misc[0];
    pdl_wait();
    pdl_release();

    uint64_t x = 0, x_end = 0;
    const AttnFound found = attn_find<C::THREADS>(p, C::ROWS, TC_KEYS, sh, [&](uint64_t total) {
        const uint32_t n = attn_ranges(total, p.ctas, p.least_tiles);
        if (blockIdx.x < n) { x = attn_range_begin(total, n, blockIdx.x); x_end = attn_range_begin(total, n, blockIdx.x + 1); }
        return x < x_end ? x : ~0ull;
    });
    AttnWalk walk(p, found, x, x_end, C::ROWS, TC_KEYS);
    // rows of a row tile of the item, the keys its last row sees, and its tiles within the piece
    auto tile_rows = [&](uint32_t g) {
        const uint32_t all = walk.sq.q_len * p.group, r0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS;
        return all > r0 ? min(all - r0, TC_TILE_ROWS) : 0u;
    };
    auto tiles_of = [&](uint32_t g) {
        const uint32_t rows = tile_rows(g);
        if (rows == 0) return 0u;
        const uint32_t keys = attn_row_keys(walk.sq, (walk.at.block * C::ROWS + g * TC_TILE_ROWS + rows - 1) / p.group);
        const uint32_t t = min(max((keys + TC_KEYS - 1) / TC_KEYS, 1u), walk.t1);
        return t > walk.t0 ? t - walk.t0 : 0u;
    };
    // tiles of the piece that any row tile wants (the last tile that has rows wants the most)
    auto tiles_wanted = [&] { return NQ == 2 ? max(tiles_of(0), tiles_of(NQ - 1)) : tiles_of(0); };

    if (warp < 4) {
        if constexpr (C::AUX_REGS < C::LAUNCH_REGS) regs_down<C::AUX_REGS>();
        if (warp == 0) {
            // ---- TMA: K and V of a tile, one lane a box ----
            const uint32_t per_tile = TC_KEYS / box_rows;
            const AttnDivisor div = attn_divisor(p.block_size);
            uint32_t ks = 0, kph = 0, vs = 0, vph = 0, tail_ph = 0, rs = 0, rph = 0;
            bool ok = true;
            while (ok && walk.next(p)) {
                const int32_t* table = p.block_table + size_t(walk.seq) * p.table_stride;
                const uint32_t n = tiles_wanted(), kv_len = walk.sq.kv_len;
                const uint32_t none = p.n_pages * p.block_size;              // a row behind the last page: TMA fills with zeros
                auto find = [&](uint32_t j) -> uint32_t {                    // cache row of this lane's box of tile j
                    const uint32_t pos = (walk.t0 + j) * TC_KEYS + lane * box_rows;
                    if (j >= n || lane >= per_tile || pos >= kv_len) return none;
                    const uint32_t page = attn_div(pos, div), id = uint32_t(table[page]);
                    if (id >= p.n_pages) { record_status(STATUS_PAGE_OUT_OF_RANGE); return none; }
                    return id * p.block_size + (pos - page * p.block_size);
                };
                uint32_t row_next = find(0);
                for (uint32_t j = 0; ok && j < n; ++j) {
                    const uint32_t row = row_next, pos0 = (walk.t0 + j) * TC_KEYS;
                    row_next = find(j + 1);
                    const uint32_t left = kv_len > pos0 ? kv_len - pos0 : 0u, boxes = min((left + box_rows - 1) / box_rows, per_tile);
                    if constexpr (!FP8) {
                        ok = mbar_wait_warp(K_EMPTY + 8 * ks, kph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                        if (!ok) break;
                        const uint32_t kd = base + C::OFF_K + ks * C::TILE;
                        if (lane == 0) mbar_arrive_expect_tx(K_FULL + 8 * ks, boxes * box_rows * 128u * C::PANELS);
                        __syncwarp();
                        if (lane < boxes)
#pragma unroll
                            for (int pn = 0; pn < C::PANELS; ++pn)
                                tma_load_3d(kd + pn * C::PANEL + lane * box_rows * 128u, &map_k, pn * 64, int32_t(walk.at.head), int32_t(row), K_FULL + 8 * ks);
                        __syncwarp();
                        if (++ks == uint32_t(ST)) { ks = 0; kph ^= 1u; }
                        ok = mbar_wait_warp(V_EMPTY + 8 * vs, vph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                        if (!ok) break;
                        const uint32_t vd = base + C::OFF_V + vs * C::TILE;
                        const bool tail = left < TC_KEYS;
                        const uint32_t full = tail ? V_TAIL : V_FULL + 8 * vs;
                        if (lane == 0) mbar_arrive_expect_tx(full, boxes * box_rows * 128u * C::PANELS);
                        __syncwarp();
                        if (lane < boxes)
#pragma unroll
                            for (int pn = 0; pn < C::PANELS; ++pn)
                                tma_load_3d(vd + pn * C::PANEL + lane * box_rows * 128u, &map_v, pn * 64, int32_t(walk.at.head), int32_t(row), full);
                        __syncwarp();
                        if (tail) {
                            // behind the sequence's end a page holds anything, and zero times a NaN is one: zeros before the product
                            ok = mbar_wait_warp(V_TAIL, tail_ph, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER);
                            tail_ph ^= 1u;
                            if (!ok) break;
                            for (uint32_t i = lane; i < (TC_KEYS - left) * 8u; i += 32)
#pragma unroll
                                for (int pn = 0; pn < C::PANELS; ++pn) sts128(vd + pn * C::PANEL + left * 128u + i * 16u, 0u, 0u, 0u, 0u);
                            fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(V_FULL + 8 * vs);
                            __syncwarp();
                        }
                        if (++vs == uint32_t(ST)) { vs = 0; vph ^= 1u; }
                    } else {
#pragma unroll 1
                        for (int side = 0; side < 2; ++side) {
                            ok = ok && mbar_wait_warp(RAW_EMPTY + 8 * rs, rph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                            if (!ok) break;
                            if (lane == 0) mbar_arrive_expect_tx(RAW_FULL + 8 * rs, boxes * box_rows * uint32_t(DP));
                            __syncwarp();
                            if (lane < boxes) {
                                const uint32_t dst = base + C::OFF_RAW + rs * C::RAW + lane * box_rows * uint32_t(DP);
                                tma_load_3d(dst, side ? &map_v : &map_k, 0, int32_t(walk.at.head), int32_t(row), RAW_FULL + 8 * rs);
                            }
                            __syncwarp();
                            if (++rs == uint32_t(C::RAW_STAGES)) { rs = 0; rph ^= 1u; }
                        }
                    }
                }
            }
        } else if (warp == 1) {
            // ---- MMA ----
            constexpr uint32_t idesc_s = attn_idesc(TC_KEYS, FP8, false), idesc_o = attn_idesc(DP, FP8, true);
            uint32_t ks = 0, kph = 0, vs = 0, vph = 0, q_ph[2] = {0, 0}, p_ph[2] = {0, 0};
            bool ok = true;
            auto scores = [&](uint32_t g, uint32_t stage) {
                if (elect_one()) {
                    const uint64_t q = make_kmajor_sw128_desc(base + C::OFF_Q + g * C::TILE), k = make_kmajor_sw128_desc(base + C::OFF_K + stage * C::TILE);
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
                        umma_bf16_ss<false>(tmem + g * 128u, q + (s >> 2) * (C::PANEL >> 4) + (s & 3) * 2, k + (s >> 2) * (C::PANEL >> 4) + (s & 3) * 2, idesc_s, s ? 1u : 0u);
                    umma_commit<false>(S_FULL + 8 * g);
                }
                __syncwarp();
            };
            while (ok && walk.next(p)) {
                const uint32_t n_g[2] = {tiles_of(0), NQ == 2 ? tiles_of(NQ - 1) : 0u}, n = max(n_g[0], n_g[1]);
                if (n == 0) continue;
                ok = mbar_wait_warp(K_FULL + 8 * ks, kph, abort_flag, STATUS_WAIT_EXPIRED_MMA, 20);
                if (!ok) break;
#pragma unroll
                for (uint32_t g = 0; g < uint32_t(NQ); ++g) {
                    if (n_g[g] == 0) continue;
                    ok = ok && mbar_wait_warp(Q_FULL + 8 * g, q_ph[g], abort_flag, STATUS_WAIT_EXPIRED_MMA, 20);
                    if (!ok) break;
                    q_ph[g] ^= 1u;
                    tcgen05_fence_after();
                    scores(g, ks);
                }
                if (!ok) break;
                if (elect_one()) umma_commit<false>(K_EMPTY + 8 * ks);
                __syncwarp();
                if (++ks == uint32_t(ST)) { ks = 0; kph ^= 1u; }
                for (uint32_t j = 0; ok && j < n; ++j) {
                    ok = mbar_wait_warp(V_FULL + 8 * vs, vph, abort_flag, STATUS_WAIT_EXPIRED_MMA, 20);
                    if (ok && j + 1 < n) ok = mbar_wait_warp(K_FULL + 8 * ks, kph, abort_flag, STATUS_WAIT_EXPIRED_MMA, 20);
                    if (!ok) break;
                    const uint32_t vd = base + C::OFF_V + vs * C::TILE;
#pragma unroll
                    for (uint32_t g = 0; g < uint32_t(NQ); ++g) {
                        if (j >= n_g[g]) continue;
                        ok = ok && mbar_wait_warp(P_FULL + 8 * g, p_ph[g], abort_flag, STATUS_WAIT_EXPIRED_MMA);
                        if (!ok) break;
                        p_ph[g] ^= 1u;
                        tcgen05_fence_after();
                        if (elect_one()) {
                            const uint64_t v = make_mnmajor_sw128_desc(vd, C::PANEL);
#pragma unroll
                            for (int s = 0; s < int(TC_KEYS) / 16; ++s)
                                umma_bf16_ts<false>(tmem + NQ * 128u + g * uint32_t(DP), tmem + g * 128u + s * 8u, v + s * (2048 >> 4), idesc_o, (j | s) ? 1u : 0u);
                            umma_commit<false>(PV_DONE + 8 * g);
                        }
                        __syncwarp();
                        if (j + 1 < n_g[g]) scores(g, ks);
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        umma_commit<false>(V_EMPTY + 8 * vs);
                        if (j + 1 < n) umma_commit<false>(K_EMPTY + 8 * ks);
                    }
                    __syncwarp();
                    if (++vs == uint32_t(ST)) { vs = 0; vph ^= 1u; }
                    if (j + 1 < n && ++ks == uint32_t(ST)) { ks = 0; kph ^= 1u; }
                }
            }
        } else {
            // ---- Q of the items ahead to L2, so that its rows' latency is that of L2 when their turn comes ----
            const uint32_t t = (warp - 2) * 32u + lane;
            while (walk.next(p)) {
                const uint32_t row0 = walk.at.block * C::ROWS, rows = tile_rows(0) + (NQ == 2 ? tile_rows(NQ - 1) : 0u), lines = (p.head_dim * 2u + 127u) / 128u;
                for (uint32_t i = t; i < rows * lines; i += 64u) {
                    const uint32_t row = row0 + i / lines, tok = row / p.group;
                    const uint16_t* at = p.q + size_t(walk.sq.row0 + tok) * p.q_row_stride + size_t(walk.at.head * p.group + row - tok * p.group) * p.head_dim + (i % lines) * 64u;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                }
            }
        }
    } else if (warp < uint32_t(C::CONV_WARP0)) {
        // ---- softmax: a row a thread ----
        if constexpr (C::SOFT_REGS > C::LAUNCH_REGS) regs_up<C::SOFT_REGS>();
        const uint32_t g = (warp - 4) >> 2, quad = warp & 3u, row_in = quad * 32u + lane;
        const uint32_t t_s = tmem + g * 128u + ((quad * 32u) << 16), t_o = tmem + NQ * 128u + g * uint32_t(DP) + ((quad * 32u) << 16);
        const uint32_t q_tile = base + C::OFF_Q + g * C::TILE;
        float* const scale_s = reinterpret_cast<float*>(gen + C::OFF_SCALE) + g * TC_TILE_ROWS;
        const uint32_t D = p.head_dim;
        const AttnDivisor group_div = attn_divisor(p.group);
        uint32_t s_ph = 0, pv_ph = 0;
        bool ok = true;
        while (ok && walk.next(p)) {
            const uint32_t n = tiles_of(g), rows = tile_rows(g);
            if (rows == 0) continue;
            const uint32_t row0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS;
            float c = p.scale * p.k_scale * ATTN_LOG2E, m = -INFINITY, l = 0.0f;
            if (n) {
                // Q: this warp's 32 rows, sixteen bytes a lane
                constexpr uint32_t CH = DP / 8;
                const uint16_t* const q_head = p.q + size_t(walk.sq.row0) * p.q_row_stride + size_t(walk.at.head) * p.group * D;
                uint4 qv[CH];                                                // (all loads in flight: one latency)
#pragma unroll
                for (uint32_t i = 0; i < CH; ++i) {
                    const uint32_t idx = i * 32u + lane, r = quad * 32u + idx / CH, ch = idx % CH, row = row0 + r, tok = attn_div(row, group_div);
                    qv[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (r < rows && ch * 8u < D) qv[i] = *reinterpret_cast<const uint4*>(q_head + size_t(tok) * p.q_row_stride + (row - tok * p.group) * D + ch * 8u);
                }
#pragma unroll
                for (uint32_t i = 0; i < CH; ++i) {
                    const uint32_t idx = i * 32u + lane, r = quad * 32u + idx / CH, ch = idx % CH;
                    uint4 v = qv[i];
                    if constexpr (FP8) {
                        uint32_t w[4] = {v.x, v.y, v.z, v.w}, top = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, (w[k] >> 16) & 0x7FFFu));
#pragma unroll
                        for (uint32_t o = 1; o < CH && o < 32u; o <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                        const int e = int(top >> 7), by = e == 0 || e == 255 ? 0 : min(max(141 - e, -120), 120);
                        const float up = __uint_as_float(uint32_t(127 + by) << 23);
                        if (ch == 0) scale_s[r] = __uint_as_float(uint32_t(127 - by) << 23);
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = pack_pair<true>(bf16_lo(w[k]) * up, bf16_hi(w[k]) * up);
                        v = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    sts128(q_tile + (ch >> 3) * C::PANEL + sw128_off(r, ch & 7u), v.x, v.y, v.z, v.w);
                }
                fence_proxy_async();
                __syncwarp();
                mbar_arrive(Q_FULL + 8 * g);
                if constexpr (FP8) c *= scale_s[row_in];
            }
            const uint32_t row = row0 + row_in, tok = attn_div(row, group_div), head = walk.at.head * p.group + row - tok * p.group;
            const uint32_t keys = row_in < rows ? attn_row_keys(walk.sq, tok) : 0u, all_see = attn_row_keys(walk.sq, row0 / p.group);
            for (uint32_t j = 0; ok && j < n; ++j) {
                ok = mbar_wait(S_FULL + 8 * g, s_ph, abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                s_ph ^= 1u;
                tcgen05_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld32(t_s + 32 * k, s + 32 * k);
                tmem_ld_wait();
                const uint32_t pos0 = (walk.t0 + j) * TC_KEYS;
                if (pos0 + TC_KEYS > all_see) {
                    const uint32_t mine = keys > pos0 ? keys - pos0 : 0u;
#pragma unroll
                    for (uint32_t k = 0; k < 128; ++k)
                        if (k >= mine) s[k] = 0xFF800000u;                   // -inf
                }
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 128; k += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) top4[u] = fmaxf(fmaxf(top4[u], __uint_as_float(s[k + 2 * u])), __uint_as_float(s[k + 2 * u + 1]));
                const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * c;
                const bool grow = top > m + (j ? TC_RESCALE : 0.0f);
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xFFFFFFFFu, grow)) {
                    // O is this thread's row until the next P is handed over, once the product before has been added
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(PV_DONE + 8 * g, pv_ph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const float keep = grow ? ex2(m - top) : 1.0f;
                    if (grow) m = top;
                    l *= keep;
#pragma unroll 1
                    for (int k = 0; k < DP; k += 16) {
                        uint32_t v[16];
                        tmem_ld16(t_o + k, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int u = 0; u < 16; ++u) v[u] = __float_as_uint(__uint_as_float(v[u]) * keep);
                        tmem_st16(t_o + k, v);
                    }
                }
                const float off = m == -INFINITY ? 0.0f : -m;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 128; k += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        const float a = ex2(fmaf(__uint_as_float(s[k + 2 * u]), c, off)), b = ex2(fmaf(__uint_as_float(s[k + 2 * u + 1]), c, off));
                        sum[u & 3] += a + b;
                        w[u] = pack_pair<FP8>(a, b);
                    }
                    tmem_st16(t_s + (k >> 1), w);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tcgen05_fence_before();
                mbar_arrive(P_FULL + 8 * g);
                pv_ph ^= 1u;
            }
            if (!ok) break;
            // ---- the piece is done ----
            const bool whole = walk.whole();
            if (n) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(PV_DONE + 8 * g, pv_ph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE));
                if (!ok) break;
                tcgen05_fence_after();
            }
            if (!whole) {
                float* part = p.parts + attn_part_floats(C::ROWS, DP) * (2 * size_t(blockIdx.x) + (walk.t0 == 0 ? 1 : 0));
                const uint32_t r = g * TC_TILE_ROWS + row_in;
#pragma unroll 1
                for (int k = 0; k < DP; k += 16) {
                    uint32_t v[16] = {};
                    if (n) { tmem_ld16(t_o + k, v); tmem_ld_wait(); }
                    if (row_in < rows)
#pragma unroll
                        for (int u = 0; u < 16; u += 4)
                            *reinterpret_cast<uint4*>(part + size_t(r) * DP + k + u) = make_uint4(v[u], v[u + 1], v[u + 2], v[u + 3]);
                }
                if (row_in < rows) { part[size_t(C::ROWS) * DP + r] = m; part[size_t(C::ROWS) * DP + C::ROWS + r] = l; }
            } else {
                // through this warp's rows of the Q tile (all of its scores have been computed), then whole rows out
                const float inv = l == 0.0f ? 0.0f : p.v_scale / l;
                bool odd = false;
#pragma unroll 1
                for (int k = 0; k < DP; k += 16) {
                    uint32_t v[16] = {}, w[8];
                    if (n) { tmem_ld16(t_o + k, v); tmem_ld_wait(); }
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const float a = l == 0.0f ? 0.0f : __uint_as_float(v[2 * u]) * inv, b = l == 0.0f ? 0.0f : __uint_as_float(v[2 * u + 1]) * inv;
                        odd |= !isfinite(a) || !isfinite(b);
                        w[u] = pack_bf16x2(a, b);
                    }
                    const uint32_t to = q_tile + (k >> 6) * C::PANEL, ch = (k >> 3) & 7u;
                    sts128(to + sw128_off(row_in, ch), w[0], w[1], w[2], w[3]);
                    sts128(to + sw128_off(row_in, ch + 1), w[4], w[5], w[6], w[7]);
                }
                if (p.lse && row_in < rows) p.lse[size_t(walk.sq.row0 + tok) * p.q_heads + head] = attn_lse(m, l);
                __syncwarp();
                constexpr uint32_t CH = DP / 8;
                uint16_t* const o_head = p.out + size_t(walk.sq.row0) * p.out_row_stride + size_t(walk.at.head) * p.group * D;
#pragma unroll 8
                for (uint32_t i = 0; i < CH; ++i) {
                    const uint32_t idx = i * 32u + lane, r = quad * 32u + idx / CH, ch = idx % CH, rw = row0 + r, t = attn_div(rw, group_div);
                    const uint4 v = lds128(q_tile + (ch >> 3) * C::PANEL + sw128_off(r, ch & 7u));
                    if (r < rows && ch * 8u < D) *reinterpret_cast<uint4*>(o_head + size_t(t) * p.out_row_stride + (rw - t * p.group) * D + ch * 8u) = v;
                }
                __syncwarp();
                uint32_t again = walk.sq.q_len > 1 ? __ballot_sync(0xFFFFFFFFu, odd && row_in < rows) : 0u;
                while (again) {
                    const uint32_t k = __ffs(again) - 1u;
                    again &= again - 1u;
                    attn_row_again(p, FP8, walk.seq, walk.sq.row0 + __shfl_sync(0xFFFFFFFFu, tok, k), __shfl_sync(0xFFFFFFFFu, head, k), __shfl_sync(0xFFFFFFFFu, keys, k));
                }
            }
            tcgen05_fence_before();                                          // O has been read before the next item's P is handed over
        }
    } else if constexpr (FP8) {
        // ---- raw tiles to FP16 ones ----
        if constexpr (C::AUX_REGS < C::LAUNCH_REGS) regs_down<C::AUX_REGS>();
        const uint32_t t = tid - 32u * C::CONV_WARP0;
        uint32_t rs = 0, rph = 0, st[2] = {0, 0}, ph[2] = {0, 0};
        bool ok = true;
        while (ok && walk.next(p)) {
            const uint32_t n = tiles_wanted(), kv_len = walk.sq.kv_len;
            for (uint32_t j = 0; ok && j < n; ++j) {
                const uint32_t pos0 = (walk.t0 + j) * TC_KEYS, left = kv_len > pos0 ? min(kv_len - pos0, TC_KEYS) : 0u;
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    ok = ok && mbar_wait(RAW_FULL + 8 * rs, rph, abort_flag, STATUS_WAIT_EXPIRED_DEQUANT) &&
                         mbar_wait((side ? V_EMPTY : K_EMPTY) + 8 * st[side], ph[side] ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_DEQUANT);
                    if (!ok) break;
                    const uint32_t raw = base + C::OFF_RAW + rs * C::RAW, to = base + (side ? C::OFF_V : C::OFF_K) + st[side] * C::TILE;
                    constexpr uint32_t CH = DP / 16;                         // 16-byte pieces of a raw row
#pragma unroll 4
                    for (uint32_t i = 0; i < CH; ++i) {
                        const uint32_t idx = i * 128u + t, r = idx / CH, ch = idx % CH;
                        uint4 v = lds128(raw + idx * 16u);
                        if (r >= left) v = make_uint4(0u, 0u, 0u, 0u);       // behind the sequence's end: what was there before, or nothing
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w[k] & 0xFFFFu), __NV_E4M3);
                            const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w[k] >> 16), __NV_E4M3);
                            h[2 * k] = uint32_t(a.x) | uint32_t(a.y) << 16;
                            h[2 * k + 1] = uint32_t(b.x) | uint32_t(b.y) << 16;
                        }
                        const uint32_t panel = to + (ch >> 2) * C::PANEL, c0 = (2u * ch) & 7u;
                        sts128(panel + sw128_off(r, c0), h[0], h[1], h[2], h[3]);
                        sts128(panel + sw128_off(r, c0 + 1u), h[4], h[5], h[6], h[7]);
                    }
                    fence_proxy_async();
                    mbar_arrive((side ? V_FULL : K_FULL) + 8 * st[side]);
                    mbar_arrive(RAW_EMPTY + 8 * rs);
                    if (++rs == uint32_t(C::RAW_STAGES)) { rs = 0; rph ^= 1u; }
                    if (++st[side] == uint32_t(ST)) { st[side] = 0; ph[side] ^= 1u; }
                }
            }
        }
    }
    // Teardown: after a wait that ran out, the copies and products in flight get time to land before shared and tensor memory go.
    __syncwarp();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 2) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace attn
}  // namespace atlas
