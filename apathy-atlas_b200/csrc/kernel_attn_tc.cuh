// Paged attention for many rows (chunks of a prompt, and few-token chunks with many heads to a KV head): tcgen05.
//
// A block is two tiles of 128 rows (DP 256: one).  A step is 64 keys: scores S = Q K^T [128 x 64], and O += P V with O [128 x DP], all in tensor
// memory, for each row tile g:
//     S_g even | S_g odd (64 columns each)  ...  O_g (DP columns each)      P_g, BF16, over the first half of its S's columns
// The scores of step u + 2 follow the product with P of step u, whose columns they take; those of step u + 1 are there already.  So the
// softmax of a row tile goes from step to step without waiting for the tensor cores, and they work on one tile's step while the other's
// is in its softmax.  (With S of 128 keys in one piece a tile's softmax, product and next scores were one chain: 3900 cycles for 128
// keys of both tiles, of which the tensor cores worked 2090.  A product of 64 columns reads 6 KB of shared memory for 32 cycles of
// arithmetic, so it takes 48: 2560 cycles is what is left of the chain.)
//
// One thread owns a row: its scores come to its registers (tcgen05.ld), maximum and sum need no exchange with other threads, P goes back
// to tensor memory as the A operand.  Q, K, V are 128-byte-swizzled tiles in shared memory: Q and K K-major, V as it lies in the cache
// ([key][channel]), the MN-major form of the B operand.  K and V come 128 keys at a time, page by page by TMA, in boxes of the largest
// power of two that divides page and tile; zero fill stands in for pages that do not exist and for channels behind head_dim.  Pages that
// no box of eight rows divides are copied row by row past the registers, by warps 0 and 2 in turn (pages of 5, 2048 tokens over 8192,
// 8 Q + 2 KV heads of 128: 118 us; the mma.sync form takes 433, pages of 16 by TMA 70).
//
// O is multiplied with 2^(M_old - M_new) only where a row's maximum has grown by more than 2^15 (TC_RESCALE) since O's last factor: until
// then the weights are 2^(s - M) with the old M, up to 2^15 and in the same FP32 sums, which is the same quotient.  (E4M3: FP16 holds 2^15, and M
// begins 2^7 below the largest, see ATTN_UP, so from 2^8 on.)  That
// takes the correction off the path of nearly every step (8192 tokens, scores' deviations from 1 to 4: 490 us with 2^8, 481 with 2^15).
// (Exponentials by a polynomial on the FMA pipe for a quarter to a half of the scores, the special-function unit being the busiest of the
// softmax: no faster.  The next step's scores asked for between the exponentials of this one: they are not there yet, 484 -> 564 us.)
//
// Warps: 0 TMA (or 0 and 2 copies), 1 and 3 MMA of a row tile each (converged, one lane issues), 2 tensor memory; 4-7 and 8-11 softmax, epilogue and Q
// of a row tile each, the next item's Q before this one's output; E4M3 caches: 12-15 turn raw tiles into FP16 ones (one instruction for
// two values, exact, NaN kept; Q as FP16 with a power of two per row, see the mma.sync form).  Every wait is bounded as elsewhere in the
// library.
#pragma once

#include "kernel_attn.cuh"
#include "kernel_tc.cuh"

namespace atlas {
namespace attn {

using namespace atlas::tc;

constexpr uint32_t TC_KEYS = 128, TC_STEP = 64, TC_TILE_ROWS = 128;
constexpr float TC_RESCALE = 15.0f;

template <int DP, bool FP8> struct TcCfg {
    static constexpr int NQ = DP <= 128 ? 2 : 1;                             // row tiles
    static constexpr int ROWS = NQ * int(TC_TILE_ROWS);
    static constexpr int PANELS = DP / 64;                                   // 128-byte panels of a row
    // Keys of a tile of K or V: two steps, or one for E4M3 rows of 256, where tiles of two leave room for a raw one, a K and a V alone (8192
    // tokens, 8 Q + 2 KV heads: 508 us, with one step 471; eight times 64 over 2000, 32 + 8 heads: 85 and 68).  BF16 rows of 256 are
    // bound by what their boxes bring (421 us, with one step 441).
    static constexpr int KEYS = DP <= 128 || !FP8 ? 128 : 64;
    static constexpr int Q_PANEL = 128 * 128, Q_TILE = PANELS * Q_PANEL;     // Q of a row tile
    static constexpr int PANEL = KEYS * 128, TILE = PANELS * PANEL;          // K or V of a key tile
    // K and V tiles share a ring, in the order the products take them (tc_turn).  A tile takes some 3000 cycles from request to
    // arrival where every SM asks for one a thousand cycles; with two stages of either side, each released with the last product of an
    // iteration, the MMA warp waited 870 cycles an iteration of 2090.
    static constexpr int SLOTS = DP <= 64 ? 8 : FP8 ? 4 : DP <= 128 ? 5 : 2;
    static constexpr int RAW = FP8 ? KEYS * DP : 0, RAW_STAGES = FP8 ? 2 : 0;
    static constexpr int OFF_Q = 0, OFF_KV = NQ * Q_TILE, OFF_RAW = OFF_KV + SLOTS * TILE;
    static constexpr int OFF_BAR = OFF_RAW + RAW_STAGES * RAW;
    static constexpr int N_BAR = 2 * SLOTS + 1 + 7 * NQ + 2 * RAW_STAGES;
    static constexpr int OFF_MISC = OFF_BAR + N_BAR * 8;                     // tensor memory, -, abort; attn_begin's words
    static constexpr int SMEM = OFF_MISC + 16 + 16 * 8 + int(sizeof(AttnStart)) + 1024;
    static constexpr int SOFT_WARPS = 4 * NQ, WARPS = 4 + SOFT_WARPS + (FP8 ? 4 : 0), THREADS = 32 * WARPS;
    static constexpr int CONV_WARP0 = 4 + SOFT_WARPS;
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
// 32 bytes of a row in one store (whole sectors)
__device__ __forceinline__ void stg256(void* to, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// Two FP32 values in one register pair and one issue slot.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void of_pair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

// What lies at turn t of a piece of n tiles: tiles of two steps K 0, V 0, K 1, V 1, ...; of one step K 0, K 1, V 0, K 2, V 1, ..., V n - 1,
// as the scores are two steps ahead of the product with P.
template <int STEPS> __device__ __forceinline__ void tc_turn(uint32_t t, uint32_t n, uint32_t& side, uint32_t& tile) {
    if constexpr (STEPS == 2) {
        side = t & 1u;
        tile = t >> 1;
    } else {
        side = t != 0u && ((t & 1u) == 0u || t == 2u * n - 1u) ? 1u : 0u;
        tile = t == 2u * n - 1u ? n - 1u : side ? (t - 2u) / 2u : (t + 1u) / 2u;
    }
}

template <int DP, bool FP8>
__global__ void __launch_bounds__(TcCfg<DP, FP8>::THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p, const uint32_t box_rows) {
    using C = TcCfg<DP, FP8>;
    constexpr int NQ = C::NQ, SLOTS = C::SLOTS, STEPS = C::KEYS / int(TC_STEP);
    constexpr uint32_t KEYS = C::KEYS;
    extern __shared__ uint8_t attn_smem_raw[];
    const uint32_t base = (smem_u32(attn_smem_raw) + 1023u) & ~1023u;
    uint8_t* const gen = attn_smem_raw + (base - smem_u32(attn_smem_raw));
    const uint32_t bar = base + C::OFF_BAR;
    const uint32_t FULL = bar, EMPTY = bar + 8 * SLOTS, V_TAIL = bar + 16 * SLOTS, Q_FULL = V_TAIL + 8,
                   S_FULL = Q_FULL + 8 * NQ, P_FULL = S_FULL + 16 * NQ, PV_DONE = P_FULL + 16 * NQ, RAW_FULL = PV_DONE + 16 * NQ, RAW_EMPTY = RAW_FULL + 8 * C::RAW_STAGES;
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(gen + C::OFF_MISC);
    volatile uint32_t* const abort_flag = misc + 2;
    uint64_t* const sh = reinterpret_cast<uint64_t*>(gen + C::OFF_MISC + 16);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

    if (tid == 0) {
        for (int i = 0; i < SLOTS; ++i) { mbar_init(FULL + 8 * i, FP8 ? 128 : 1); mbar_init(EMPTY + 8 * i, NQ); }
        mbar_init(V_TAIL, 1);
        for (int g = 0; g < NQ; ++g) mbar_init(Q_FULL + 8 * g, 128);
        // Scores, weights and products of even and of odd steps have barriers of their own: whoever waits for one of step u knows that step
        // u - 2 is over, so a phase cannot be mistaken for the one before last.
        for (int i = 0; i < 2 * NQ; ++i) { mbar_init(S_FULL + 8 * i, 1); mbar_init(P_FULL + 8 * i, 128); mbar_init(PV_DONE + 8 * i, 1); }
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

    AttnStart* const start = reinterpret_cast<AttnStart*>(sh + C::WARPS);
    attn_begin<C::THREADS>(p, sh, start);
    AttnWalk walk(*start);
    // rows of a row tile of the item, and the steps that it takes of the piece
    auto tile_rows = [&](uint32_t g) {
        const uint32_t all = walk.sq.q_len * p.group, r0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS;
        return all > r0 ? min(all - r0, TC_TILE_ROWS) : 0u;
    };
    auto steps_of = [&](uint32_t g) {
        const uint32_t rows = tile_rows(g);
        if (rows == 0) return 0u;
        const uint32_t keys = attn_row_keys(walk.sq, attn_div(walk.at.block * C::ROWS + g * TC_TILE_ROWS + rows - 1, p.group_div));
        const uint32_t t = min(max((keys + TC_STEP - 1) / TC_STEP, 1u), 2u * walk.t1);
        return t > 2u * walk.t0 ? t - 2u * walk.t0 : 0u;
    };
    // key tiles of the piece that any row tile wants (the last row tile that has rows wants the most)
    auto tiles_wanted = [&] { return ((NQ == 2 ? max(steps_of(0), steps_of(NQ - 1)) : steps_of(0)) + STEPS - 1u) / STEPS; };

    // Tiles row by row, where no box of eight rows divides a page; a row that is not there is zeros.  Two warps, for the even and the odd
    // turns: of a ring of two places or more, so that a wait is never two phases of its barrier ahead.
    auto gather = [&](uint32_t odd) {
        constexpr uint32_t SIZE = FP8 ? 1 : 2, CH = DP * SIZE / 16, RING = FP8 ? C::RAW_STAGES : SLOTS;      // 16-byte pieces of a row
        const uint32_t EMPTY_OF = FP8 ? RAW_EMPTY : EMPTY, FULL_OF = FP8 ? RAW_FULL : FULL, bytes = p.head_dim * SIZE;
        uint32_t turn = odd;                                                 // of the CTA
        bool ok = true;
        while (ok && walk.next(p)) {
            const int32_t* table = p.block_table + size_t(walk.seq) * p.table_stride;
            const uint32_t n = tiles_wanted(), kv_len = walk.sq.kv_len;
            for (uint32_t t = odd; ok && t < 2u * n; t += 2, turn += 2) {
                uint32_t side, j;
                tc_turn<STEPS>(t, n, side, j);
                const uint32_t pos0 = walk.t0 * TC_KEYS + j * KEYS, at = turn % RING;
                int32_t rows[KEYS / 32];
#pragma unroll
                for (uint32_t k = 0; k < KEYS / 32; ++k) {
                    const uint32_t pos = pos0 + 32u * k + lane;
                    rows[k] = pos < kv_len ? attn_cache_row(p, table, pos) : -1;
                }
                const uint8_t* const cache = side ? p.v_cache : p.k_cache;
                ok = mbar_wait_warp(EMPTY_OF + 8 * at, ((turn / RING) & 1u) ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                if (!ok) break;
                const uint32_t dst = FP8 ? base + C::OFF_RAW + at * C::RAW : base + C::OFF_KV + at * C::TILE;
#pragma unroll
                for (uint32_t k = 0; k < KEYS / 32; ++k)
#pragma unroll 8
                    for (uint32_t i = 0; i < CH; ++i) {
                        const uint32_t in = i * (32u / CH) + lane / CH, r = 32u * k + in, ch = lane % CH;
                        const int32_t row = __shfl_sync(0xFFFFFFFFu, rows[k], in);
                        const bool there = row >= 0 && ch * 16u < bytes;
                        const uint8_t* from = there ? cache + (size_t(row) * p.kv_heads + walk.at.head) * bytes + ch * 16u : cache;
                        cp_async_16_zfill(FP8 ? dst + r * uint32_t(DP) + ch * 16u : dst + (ch >> 3) * C::PANEL + sw128_off(r, ch & 7u), from, there ? 16u : 0u);
                    }
                cp_async_commit();
                cp_async_wait_group<0>();
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(FULL_OF + 8 * at);
                __syncwarp();
            }
        }
    };

    if (warp < 4) {
        if (box_rows < 8u && (warp == 0 || warp == 2)) {
            gather(warp >> 1);
        } else if (warp == 0) {
            // ---- TMA: K and V of a tile, one lane a box ----
            const uint32_t per_tile = KEYS / box_rows;
            const AttnDivisor div = p.page_div;
            uint32_t slot = 0, ph = 0, tail_ph = 0, rs = 0, rph = 0;
            bool ok = true;
            while (ok && walk.next(p)) {
                const int32_t* table = p.block_table + size_t(walk.seq) * p.table_stride;
                const uint32_t n = tiles_wanted(), kv_len = walk.sq.kv_len;
                const uint32_t none = p.n_pages * p.block_size;              // a row behind the last page: TMA fills with zeros
                auto page_of = [&](uint32_t t) -> uint32_t {                 // this lane's box at turn t: its page, as the table has it
                    uint32_t side, j;
                    tc_turn<STEPS>(t, n, side, j);
                    const uint32_t pos = walk.t0 * TC_KEYS + j * KEYS + lane * box_rows;
                    return t < 2u * n && lane < per_tile && pos < kv_len ? uint32_t(table[attn_div(pos, div)]) : 0u;
                };
                uint32_t id_next = page_of(0), row = 0, left = 0, boxes = 0;
#pragma unroll STEPS
                for (uint32_t t = 0; ok && t < 2u * n; ++t) {
                    uint32_t side, j;
                    tc_turn<STEPS>(t, n, side, j);
                    if (STEPS == 1 || side == 0) {                           // (V 0 lies where K 0 lies, and comes next)
                        const uint32_t id = id_next, pos0 = walk.t0 * TC_KEYS + j * KEYS, pos = pos0 + lane * box_rows;
                        id_next = page_of(t + STEPS);
                        row = id * p.block_size + (pos - attn_div(pos, div) * p.block_size);
                        if (id >= p.n_pages) {
                            record_status(STATUS_PAGE_OUT_OF_RANGE);
                            row = none;
                        }
                        left = kv_len > pos0 ? kv_len - pos0 : 0u;
                        boxes = min((left + box_rows - 1) / box_rows, per_tile);
                    }
                    const CUtensorMap* const map = side ? &map_v : &map_k;
                    if constexpr (!FP8) {
                        ok = mbar_wait_warp(EMPTY + 8 * slot, ph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                        if (!ok) break;
                        const uint32_t dst = base + C::OFF_KV + slot * C::TILE;
                        const bool tail = side == 1 && left < KEYS;
                        const uint32_t full = tail ? V_TAIL : FULL + 8 * slot;
                        if (lane == 0) mbar_arrive_expect_tx(full, boxes * box_rows * 128u * C::PANELS);
                        __syncwarp();
                        if (lane < boxes)
#pragma unroll
                            for (int pn = 0; pn < C::PANELS; ++pn)
                                tma_load_3d(dst + pn * C::PANEL + lane * box_rows * 128u, map, pn * 64, int32_t(walk.at.head), int32_t(row), full);
                        __syncwarp();
                        if (tail) {
                            // behind the sequence's end a page holds anything, and zero times a NaN is one: zeros before the product
                            ok = mbar_wait_warp(V_TAIL, tail_ph, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER);
                            tail_ph ^= 1u;
                            if (!ok) break;
                            for (uint32_t i = lane; i < (KEYS - left) * 8u; i += 32)
#pragma unroll
                                for (int pn = 0; pn < C::PANELS; ++pn) sts128(dst + pn * C::PANEL + left * 128u + i * 16u, 0u, 0u, 0u, 0u);
                            fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(FULL + 8 * slot);
                            __syncwarp();
                        }
                        if (++slot == uint32_t(SLOTS)) { slot = 0; ph ^= 1u; }
                    } else {
                        ok = mbar_wait_warp(RAW_EMPTY + 8 * rs, rph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_PRODUCER, 20);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(RAW_FULL + 8 * rs, boxes * box_rows * uint32_t(DP));
                        __syncwarp();
                        if (lane < boxes) {
                            const uint32_t dst = base + C::OFF_RAW + rs * C::RAW + lane * box_rows * uint32_t(DP);
                            tma_load_3d(dst, map, 0, int32_t(walk.at.head), int32_t(row), RAW_FULL + 8 * rs);
                        }
                        __syncwarp();
                        if (++rs == uint32_t(C::RAW_STAGES)) { rs = 0; rph ^= 1u; }
                    }
                }
            }
        } else if (warp == 1 || (NQ == 2 && warp == 3)) {
            // ---- MMA of row tile 0 or 1: either warp waits for its own softmax only, and while it does the tensor cores have the other's work.
            // (One warp for both, in turn: 2090 cycles a step, of which 700 went by between its waits and the next product.)
            constexpr uint32_t idesc_s = attn_idesc(TC_STEP, FP8, false), idesc_o = attn_idesc(DP, FP8, true);
            const uint32_t g = warp >> 1, t_s = tmem + g * 128u, t_o = tmem + NQ * 128u + g * uint32_t(DP);
            uint32_t slot = 0, ph = 0, q_ph = 0, p_ph[2] = {0, 0};
            bool ok = true;
            auto advance = [&] { if (++slot == uint32_t(SLOTS)) { slot = 0; ph ^= 1u; } };
            auto tile_there = [&] { return mbar_wait_warp(FULL + 8 * slot, ph, abort_flag, STATUS_WAIT_EXPIRED_MMA, 20); };
            // (also for a tile that this row tile has no use for: it has been waited for, so the arrival is this round's)
            auto release = [&](uint32_t which) {
                if (elect_one()) umma_commit<false>(EMPTY + 8 * which);
                __syncwarp();
            };
            auto scores = [&](uint32_t h) {                                  // of half h of the key tile in `slot`
                if (elect_one()) {
                    const uint64_t q = make_kmajor_sw128_desc(base + C::OFF_Q + g * C::Q_TILE);
                    const uint64_t k = make_kmajor_sw128_desc(base + C::OFF_KV + slot * C::TILE + (STEPS == 2 ? h * (TC_STEP * 128u) : 0u));
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
                        umma_bf16_ss<false>(t_s + h * TC_STEP, q + (s >> 2) * (C::Q_PANEL >> 4) + (s & 3) * 2, k + (s >> 2) * (C::PANEL >> 4) + (s & 3) * 2, idesc_s, s ? 1u : 0u);
                    umma_commit<false>(S_FULL + 8 * (2 * g + h));
                }
                __syncwarp();
            };
            auto product = [&](uint32_t v_at, uint32_t u, uint32_t h) {      // of step u's P with the V at v_at
                if (elect_one()) {
                    const uint64_t v = make_mnmajor_sw128_desc(v_at, C::PANEL);
#pragma unroll
                    for (int s = 0; s < int(TC_STEP) / 16; ++s)
                        umma_bf16_ts<false>(t_o, t_s + h * TC_STEP + s * 8u, v + s * (2048 >> 4), idesc_o, (u | s) ? 1u : 0u);
                    umma_commit<false>(PV_DONE + 8 * (2 * g + h));
                }
                __syncwarp();
            };
            while (ok && walk.next(p)) {
                const uint32_t mine = steps_of(g), n = uint32_t(STEPS) * tiles_wanted();
                if (n == 0) continue;
                ok = tile_there();
                if (ok && mine) ok = mbar_wait_warp(Q_FULL + 8 * g, q_ph, abort_flag, STATUS_WAIT_EXPIRED_MMA, 20);
                if (!ok) break;
                if (mine) {
                    q_ph ^= 1u;
                    tcgen05_fence_after();
                    scores(0);
                    if (STEPS == 2 && mine > 1) scores(1);
                }
                release(slot);
                advance();
                if (STEPS == 1 && mine > 1) {
                    ok = tile_there();
                    if (!ok) break;
                    scores(1);
                    release(slot);
                    advance();
                }
                for (uint32_t u = 0; STEPS == 1 && ok && u < n; ++u) {       // (one row tile: mine is n)
                    const uint32_t h = u & 1u;
                    ok = tile_there() && mbar_wait_warp(P_FULL + 8 * (2 * g + h), p_ph[h], abort_flag, STATUS_WAIT_EXPIRED_MMA);
                    if (!ok) break;
                    p_ph[h] ^= 1u;
                    tcgen05_fence_after();
                    product(base + C::OFF_KV + slot * C::TILE, u, h);
                    release(slot);
                    advance();
                    if (u + 2 < n) {
                        ok = tile_there();
                        if (!ok) break;
                        scores(h);
                        release(slot);
                        advance();
                    }
                }
                for (uint32_t u0 = 0; STEPS == 2 && ok && u0 < n; u0 += 2) {
                    ok = tile_there();
                    if (!ok) break;
                    const uint32_t v_slot = slot, vd = base + C::OFF_KV + slot * C::TILE;
                    bool k_there = false;
                    advance();
                    if (u0 >= mine) release(v_slot);
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        const uint32_t u = u0 + h;
                        if (!ok || u >= mine) continue;
                        ok = mbar_wait_warp(P_FULL + 8 * (2 * g + h), p_ph[h], abort_flag, STATUS_WAIT_EXPIRED_MMA);
                        if (!ok) continue;
                        p_ph[h] ^= 1u;
                        tcgen05_fence_after();
                        product(vd + h * (TC_STEP * 128u), u, h);
                        if (h == 1 || u + 1 == mine) release(v_slot);
                        if (u + 2 < mine) {
                            if (!k_there) ok = tile_there();
                            if (!ok) continue;
                            k_there = true;
                            scores(h);
                        }
                    }
                    if (ok && u0 + 2 < n) {
                        if (!k_there) ok = tile_there();
                        if (!ok) break;
                        release(slot);
                        advance();
                    }
                }
            }
        }
    } else if (warp < uint32_t(C::CONV_WARP0)) {
        // ---- softmax: a row a thread ----
        const uint32_t g = (warp - 4) >> 2, quad = warp & 3u, row_in = quad * 32u + lane;
        const uint32_t t_s = tmem + g * 128u + ((quad * 32u) << 16), t_o = tmem + NQ * 128u + g * uint32_t(DP) + ((quad * 32u) << 16);
        const uint32_t q_tile = base + C::OFF_Q + g * C::Q_TILE;
        const uint32_t D = p.head_dim;
        const AttnDivisor group_div = p.group_div;
        uint32_t s_ph[2] = {0, 0};                                           // of the next step's barriers, and of the ones after
        // Q of the item that the walk is at: this warp's 32 rows, copied past the registers sixteen bytes a lane.  (The item before has had its
        // last scores computed.)  The rows of the item after it are asked for from L2, a token's heads at a time.  (By a warp of their
        // own, a line a lane and all items at once, they stood in front of the first item's rows: 4 to 20 thousand cycles.)
        float next_scale = 1.0f;                                             // E4M3: takes this row's power of two back
        auto load_q = [&] {
            const uint32_t rows = tile_rows(g), row0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS;
            if (rows == 0 || steps_of(g) == 0) return;
            constexpr uint32_t CH = DP / 8;
            const uint16_t* const q_head = p.q + size_t(walk.sq.row0) * p.q_row_stride + size_t(walk.at.head) * p.group * D;
#pragma unroll 2
            for (uint32_t i = 0; i < CH; ++i) {
                const uint32_t idx = i * 32u + lane, r = quad * 32u + idx / CH, ch = idx % CH, row = row0 + r, tok = attn_div(row, group_div);
                const bool there = r < rows && ch * 8u < D;
                cp_async_16_zfill(q_tile + (ch >> 3) * C::Q_PANEL + sw128_off(r, ch & 7u),
                                  there ? q_head + size_t(tok) * p.q_row_stride + (row - tok * p.group) * D + ch * 8u : p.q, there ? 16u : 0u);
            }
            cp_async_commit();
            AttnWalk ahead = walk;
            if (ahead.next(p)) {
                const uint32_t r0 = ahead.at.block * C::ROWS + g * TC_TILE_ROWS + quad * 32u, all = ahead.sq.q_len * p.group;
                if (r0 < all) {
                    const uint32_t tok = attn_div(r0, group_div) + lane;
                    if (tok <= attn_div(min(r0 + 31u, all - 1u), group_div))
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                                     ::"l"(p.q + size_t(ahead.sq.row0 + tok) * p.q_row_stride + size_t(ahead.at.head) * p.group * D), "r"(p.group * D * 2u) : "memory");
                }
            }
            cp_async_wait_group<0>();
            __syncwarp();
            if constexpr (FP8) {
                // FP16, by the power of two that brings the row's largest value to [2^14, 2^15); a thread has its row
                const uint32_t mine = q_tile + row_in * 128u, turn = row_in & 7u;
                uint32_t top = 0;
#pragma unroll 4
                for (uint32_t ch = 0; ch < CH; ++ch) {
                    const uint4 v = lds128(mine + (ch >> 3) * C::Q_PANEL + (((ch & 7u) ^ turn) << 4));
                    const uint32_t a = v.x & 0x7FFF7FFFu, b = v.y & 0x7FFF7FFFu, c = v.z & 0x7FFF7FFFu, d = v.w & 0x7FFF7FFFu;
                    top = __vmaxu2(top, __vmaxu2(__vmaxu2(a, b), __vmaxu2(c, d)));
                }
                top = max(top & 0xFFFFu, top >> 16);
                const int e = int(top >> 7), by = e == 0 || e == 255 ? 0 : min(max(141 - e, -120), 120);
                const float up = __uint_as_float(uint32_t(127 + by) << 23);
                next_scale = __uint_as_float(uint32_t(127 - by) << 23);
#pragma unroll 4
                for (uint32_t ch = 0; ch < CH; ++ch) {
                    const uint32_t at = mine + (ch >> 3) * C::Q_PANEL + (((ch & 7u) ^ turn) << 4);
                    const uint4 v = lds128(at);
                    sts128(at, pack_pair<true>(bf16_lo(v.x) * up, bf16_hi(v.x) * up), pack_pair<true>(bf16_lo(v.y) * up, bf16_hi(v.y) * up),
                           pack_pair<true>(bf16_lo(v.z) * up, bf16_hi(v.z) * up), pack_pair<true>(bf16_lo(v.w) * up, bf16_hi(v.w) * up));
                }
            }
            fence_proxy_async();
            __syncwarp();
            mbar_arrive(Q_FULL + 8 * g);
        };
        bool ok = true, more = walk.next(p), some_odd = false;
        if (more) load_q();
        while (ok && more) {
            // this item, as the walk goes on to the next one before its output is written
            const uint32_t n = steps_of(g), rows = tile_rows(g), row0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS, seq = walk.seq, t0 = walk.t0, seq_row0 = walk.sq.row0;
            const bool whole = walk.whole();
            const uint32_t row = row0 + row_in, tok = attn_div(row, group_div), head = walk.at.head * p.group + row - tok * p.group;
            const uint32_t keys = row_in < rows ? attn_row_keys(walk.sq, tok) : 0u, all_see = attn_row_keys(walk.sq, attn_div(row0, group_div));
            float c = p.scale * p.k_scale * ATTN_LOG2E, m = -INFINITY, l = 0.0f;
            if constexpr (FP8) c = attn_factor(c * next_scale);
            const uint64_t c2 = pair_of(c, c);
#pragma unroll 1
            for (uint32_t u = 0; ok && u < n; ++u) {
                const uint32_t h = u & 1u, t_h = t_s + h * TC_STEP;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(S_FULL + 8 * (2 * g + h), s_ph[0], abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE));
                if (!ok) break;
                {                                                            // (the two barriers take turns, and so do their phases)
                    const uint32_t t = s_ph[0] ^ 1u;
                    s_ph[0] = s_ph[1];
                    s_ph[1] = t;
                }
                tcgen05_fence_after();
                uint32_t s[TC_STEP];
                tmem_ld32(t_h, s);
                tmem_ld32(t_h + 32, s + 32);
                tmem_ld_wait();
                const uint32_t pos0 = t0 * TC_KEYS + u * TC_STEP;
                if (pos0 + TC_STEP > all_see) {
                    const uint32_t mine = keys > pos0 ? keys - pos0 : 0u;
#pragma unroll
                    for (uint32_t k = 0; k < TC_STEP; ++k)
                        if (k >= mine) s[k] = 0xFF800000u;                   // -inf
                }
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (uint32_t k = 0; k < TC_STEP; k += 8)
#pragma unroll
                    for (int v = 0; v < 4; ++v) top4[v] = fmaxf(fmaxf(top4[v], __uint_as_float(s[k + 2 * v])), __uint_as_float(s[k + 2 * v + 1]));
                const float top = attn_base<FP8>(fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])), c);
                const bool grow = top > m + (FP8 ? TC_RESCALE - ATTN_UP : TC_RESCALE);   // (weights up to 2^15 either way)
                if (u == 0) {
                    m = top;
                } else if (__any_sync(0xFFFFFFFFu, grow)) {
                    // O is this thread's row until this step's P is handed over, once the product before has been added
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(PV_DONE + 8 * (2 * g + (h ^ 1u)), s_ph[0] ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const float keep = grow ? attn_exp2(m - top) : 1.0f;
                    if (grow) m = top;
                    l *= keep;
#pragma unroll 1
                    for (int k = 0; k < DP; k += 16) {
                        uint32_t v[16];
                        tmem_ld16(t_o + k, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
                        tmem_st16(t_o + k, v);
                    }
                }
                const float off = m == -INFINITY ? 0.0f : -m;
                const uint64_t off2 = pair_of(off, off);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (uint32_t k = 0; k < TC_STEP / 32; ++k) {
                    uint32_t w[16];
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const uint64_t x2 = fma2(pair_of(__uint_as_float(s[32 * k + 2 * v]), __uint_as_float(s[32 * k + 2 * v + 1])), c2, off2);
                        float e0, e1;
                        of_pair(x2, e0, e1);
                        e0 = attn_exp2(e0);
                        e1 = attn_exp2(e1);
                        sum[v & 1] = add2(sum[v & 1], pair_of(e0, e1));
                        w[v] = pack_pair<FP8>(e0, e1);
                    }
                    tmem_st16(t_h + 16 * k, w);
                }
                {
                    float a0, a1;
                    of_pair(add2(sum[0], sum[1]), a0, a1);
                    l += a0 + a1;
                }
                tmem_st_wait();
                tcgen05_fence_before();
                mbar_arrive(P_FULL + 8 * (2 * g + h));
            }
            if (!ok) break;
            const uint32_t last_ph = s_ph[1] ^ 1u;
            if (n & 1u) { const uint32_t t = s_ph[0]; s_ph[0] = s_ph[1]; s_ph[1] = t; }    // the next item begins with the even barrier
            // ---- the piece is done: the next item's Q, then this one's output ----
            more = walk.next(p);
            if (more) load_q();
            if (rows == 0) continue;
            if (n) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(PV_DONE + 8 * (2 * g + ((n - 1u) & 1u)), last_ph, abort_flag, STATUS_WAIT_EXPIRED_EPILOGUE));
                if (!ok) break;
                tcgen05_fence_after();
            }
            if (!whole) {
                float* part = p.parts + attn_part_floats(C::ROWS, DP) * (2 * size_t(blockIdx.x) + (t0 == 0 ? 1 : 0));
                const uint32_t r = g * TC_TILE_ROWS + row_in;
#pragma unroll 1
                for (int k = 0; k < DP; k += 32) {
                    uint32_t v[32] = {};
                    if (n) { tmem_ld32(t_o + k, v); tmem_ld_wait(); }
                    if (row_in < rows)
#pragma unroll
                        for (int e = 0; e < 32; e += 8) stg256(part + size_t(r) * DP + k + e, v + e);
                }
                if (row_in < rows) { part[size_t(C::ROWS) * DP + r] = m; part[size_t(C::ROWS) * DP + C::ROWS + r] = l; }
            } else {
                const float inv = l == 0.0f ? 0.0f : p.v_scale / l;
                uint16_t* const o_row = p.out + size_t(seq_row0 + tok) * p.out_row_stride + size_t(head) * D;
                const bool wide = (reinterpret_cast<uintptr_t>(o_row) & 31u) == 0u;
                bool odd = false;
#pragma unroll 1
                for (uint32_t k = 0; k < D; k += 32) {                       // (head_dim is a multiple of 32)
                    uint32_t v[32] = {}, w[16];
                    if (n) { tmem_ld32(t_o + k, v); tmem_ld_wait(); }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float a = l == 0.0f ? 0.0f : __uint_as_float(v[2 * e]) * inv, b = l == 0.0f ? 0.0f : __uint_as_float(v[2 * e + 1]) * inv;
                        odd |= !isfinite(a) || !isfinite(b);
                        w[e] = pack_bf16x2(a, b);
                    }
                    if (row_in < rows) {
                        if (wide) {
                            stg256(o_row + k, w);
                            stg256(o_row + k + 16, w + 8);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; e += 4) *reinterpret_cast<uint4*>(o_row + k + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
                        }
                    }
                }
                if (p.lse && row_in < rows) p.lse[size_t(seq_row0 + tok) * p.q_heads + head] = attn_lse(m, l);
                some_odd |= __any_sync(0xFFFFFFFFu, odd && row_in < rows);
            }
            tcgen05_fence_before();                                          // O has been read before the next item's P is handed over
        }
        // Rows that came out not finite (see attn_row_again), once nobody waits for this warp any more: they can take longer than a wait may.
        if (ok && some_odd) {
            walk = AttnWalk(*start);
            while (walk.next(p)) {
                const uint32_t rows = tile_rows(g), row0 = walk.at.block * C::ROWS + g * TC_TILE_ROWS + quad * 32u;
                if (!walk.whole() || rows <= quad * 32u) continue;
                const uint32_t keys0 = attn_row_keys(walk.sq, attn_div(row0, group_div)), kv_len = walk.sq.kv_len;
                if (!attn_odd_values(p, FP8, walk.seq, walk.at.head, keys0, min(kv_len, keys0 + ATTN_MASKED_MOST))) continue;
                for (uint32_t r = 0; r < min(rows - quad * 32u, 32u); ++r) {
                    const uint32_t row = row0 + r, tok = attn_div(row, group_div), head = walk.at.head * p.group + row - tok * p.group;
                    const uint16_t* const o_row = p.out + size_t(walk.sq.row0 + tok) * p.out_row_stride + size_t(head) * D;
                    bool odd = false;
                    for (uint32_t d = lane; d < D; d += 32) odd |= (o_row[d] & 0x7F80u) == 0x7F80u;
                    if (__any_sync(0xFFFFFFFFu, odd)) attn_row_again<FP8>(p, walk.seq, walk.sq.row0 + tok, head, attn_row_keys(walk.sq, tok), kv_len);
                }
            }
        }
    } else if constexpr (FP8) {
        // ---- raw tiles to FP16 ones ----
        const uint32_t t = tid - 32u * C::CONV_WARP0;
        uint32_t rs = 0, rph = 0, slot = 0, ph = 0;
        bool ok = true;
        while (ok && walk.next(p)) {
            const uint32_t n = tiles_wanted(), kv_len = walk.sq.kv_len;
            for (uint32_t turn = 0; ok && turn < 2u * n; ++turn) {
                uint32_t side, j;
                tc_turn<STEPS>(turn, n, side, j);
                const uint32_t pos0 = walk.t0 * TC_KEYS + j * KEYS, left = kv_len > pos0 ? min(kv_len - pos0, KEYS) : 0u;
                ok = mbar_wait(RAW_FULL + 8 * rs, rph, abort_flag, STATUS_WAIT_EXPIRED_DEQUANT) &&
                     mbar_wait(EMPTY + 8 * slot, ph ^ 1u, abort_flag, STATUS_WAIT_EXPIRED_DEQUANT);
                if (!ok) break;
                const uint32_t raw = base + C::OFF_RAW + rs * C::RAW, to = base + C::OFF_KV + slot * C::TILE;
                constexpr uint32_t CH = DP / 16;                             // 16-byte pieces of a raw row
#pragma unroll 4
                for (uint32_t i = 0; i < KEYS * CH / 128u; ++i) {
                    const uint32_t idx = i * 128u + t, r = idx / CH, ch = idx % CH;
                    uint4 v = lds128(raw + idx * 16u);
                    if (r >= left) v = make_uint4(0u, 0u, 0u, 0u);           // behind the sequence's end: what was there before, or nothing
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
                mbar_arrive(FULL + 8 * slot);
                mbar_arrive(RAW_EMPTY + 8 * rs);
                if (++rs == uint32_t(C::RAW_STAGES)) { rs = 0; rph ^= 1u; }
                if (++slot == uint32_t(SLOTS)) { slot = 0; ph ^= 1u; }
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
