// Products of quantised rows with one quantised weight per group of rows, and an epilogue, for sm_100a:
//
//     out[i, :] = act(Q(x[i, :]) * dequant(W[g])^T + bias[g]) (* or + extra[i, :]),   offsets[g] <= i < offsets[g + 1]
//
// x is quantised to MXFP (32-element blocks along K), W is an MXFP tensor [groups, N, K]; a plain linear is one group.
// Both operands stay quantised up to the tensor cores (tcgen05.mma, block-scaled kinds).
//
// The weight is the instruction's left operand (its 128 rows are output features) and the rows of x the right one.
// The right operand's width is free in steps of 16, so a ragged group is cut into tiles of equal width and at most 15
// rows of padding, and one row costs a tile of 16 and not one of 128.  What that asks for:
//   * the rows' codes are loaded by TMA in boxes of 64 and 16 rows from the row the group begins at, whatever it is;
//   * the rows' scales are written by the quantiser in the 512-byte chunks that tcgen05.cp expects, chunks per row tile:
//     the quantiser finds its row's group and tile by itself;
//   * an accumulator holds a feature per lane and a row per column: bias is one value per lane, and the 32 lanes of a
//     warp read the second operand and write the result 32 consecutive features at a time.
// Which rows belong to which group is read on the device: no size but the upper bounds is known to the host.
//
// Operand layout in HBM:
//   weights: blocks of 128 features x one step of K, see WeightTile in mxq_grouped.cuh;
//   rows:    codes [rows, K], scales [tile slot][ceil(K / 128)][chunks][512] bytes.  With tiles of at most `width` rows, tile t of a
//            group that begins at row f has slot f / width + group + t: no two tiles share one, and no sum over the groups before is needed.
//
// Measured (replays in a row, quantiser included): 8192 rows, 4096 -> 14336, E4M3, silu and multiplier: 460 to 480 us for the first calls, 515 to 540 us run for
// seconds (1.8 PFLOP/s at 1.37 GHz under the power cap; the tensor pipe is active for 54 % of the cycles, what idles it for the rest is not known);
// 192 rows, 4096 -> 4096: 19.1 us; 8192 rows over 32 experts, 2048 -> 2048, E2M1: 65 us.
#include <algorithm>

#include "mxq_grouped.cuh"

namespace mxq {
namespace grouped {

constexpr int FIRST_EPI_WARP = 4;                // warps 0, 1, 3: weight copies, MMA issuer, row copies

// Three epilogue warps per lane quadrant (EPI_SIDES) keep up with tall tiles (8192 rows, 32 experts of 2048 x 2048 in four bits: 70.8 -> 65.3 us
// against two); narrow ones take two, and the shared memory as one more stage (192 x 4096 x 4096: 19.7 -> 19.1).
// A CTA's tile is 128 features x at most BT rows; MXF4: both operands packed E2M1 nibbles (256 elements of K per 128 bytes).
// CTAS = 2: a pair of CTAs on two neighbouring SMs takes 256 features and the same rows, each brings its own weights and half of the
// rows: what tensor tiles read from L2 bounds a large product, and a pair reads two thirds (32 KB a step and SM instead of 48).
template <int BT_, int STAGES_, bool MXF4_, int CTAS_, int EPI_SIDES_> struct Cfg {
    static constexpr int BT = BT_, STAGES = STAGES_, CTAS = CTAS_;
    static constexpr bool MXF4 = MXF4_;
    static constexpr int EPI_SIDES = EPI_SIDES_, EPI_WARPS = 4 * EPI_SIDES, THREADS = (FIRST_EPI_WARP + EPI_WARPS) * 32;
    static constexpr int FEATURES = 128 * CTAS;                     // of a unit of work
    using Tile = WeightTile<MXF4>;
    static constexpr int K_STEP = Tile::K_STEP, SF_STEPS = Tile::SF_STEPS;          // elements of K and 128-element steps of scales per stage
    static constexpr int X_BYTES = BT / CTAS * 128, X_CHUNKS = BT > 128 ? 2 : 1;
    // a stage: weight codes | row codes | scales: [SF_STEPS][512] of the weights, [SF_STEPS][X_CHUNKS][512] of the rows; in a pair the
    // weights' scales lie behind their codes, as in memory: one copy brings both
    static constexpr int X = CTAS == 2 ? (Tile::BYTES + 1023) / 1024 * 1024 : Tile::CODES, SFW = CTAS == 2 ? Tile::CODES : X + X_BYTES;
    static constexpr int SFX = CTAS == 2 ? X + X_BYTES : SFW + SF_STEPS * 512;
    static constexpr int STAGE_BYTES = (SFX + SF_STEPS * X_CHUNKS * 512 + 1023) / 1024 * 1024;      // the 128-byte swizzle repeats every 1024 bytes
    // Two accumulators of BT columns, tiles in turn: one is read while the next is computed.  Behind them two sets of scale columns.
    static constexpr int ACC_STRIDE = BT > 128 ? 256 : BT;
    static constexpr int SF_COLS = SF_STEPS * 8;
    static constexpr int SFW_COL = BT > 128 ? BT : 2 * ACC_STRIDE, SFX_COL = BT > 128 ? ACC_STRIDE + BT : SFW_COL + 2 * SF_COLS;
    static_assert(BT <= 128 || BT + 2 * SF_COLS <= ACC_STRIDE, "tensor memory");
    static_assert(SFX_COL + 2 * SF_COLS <= 512, "tensor memory");
    // behind the ring: barriers, the group table, the epilogue's 2 KiB per warp
    static constexpr int TABLE_END = (256 + 2 * (MAX_GROUPS + 1) * 4 + 15) / 16 * 16;
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + TABLE_END + EPI_WARPS * 2048;
    static_assert(SMEM_BYTES <= 232448, "more shared memory than a CTA can have");
};
using Narrow = Cfg<128, 6, false, 1, 2>;
using NarrowFp4 = Cfg<128, 5, true, 1, 2>;
using Tall = Cfg<240, 4, false, 1, 3>;
using TallFp4 = Cfg<224, 4, true, 1, 3>;
using Pair = Cfg<240, 5, false, 2, 3>;
using PairFp4 = Cfg<224, 5, true, 2, 3>;

template <class C, int DT>
__global__ void __launch_bounds__(C::THREADS, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_x64, const __grid_constant__ CUtensorMap map_x16, const __grid_constant__ CUtensorMap map_x8,
               const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sf, const __grid_constant__ Params p) {
    constexpr int STAGES = C::STAGES, CTAS = C::CTAS, EPI_SIDES = C::EPI_SIDES, EPI_WARPS = C::EPI_WARPS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw);
    const uint32_t bars = ring + STAGES * C::STAGE_BYTES;            // full[S], empty[S], accum_full[2], accum_empty[2], drain, tmem slot
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring_ptr + STAGES * C::STAGE_BYTES + 8 * (2 * STAGES + 5));
    int* tiles = reinterpret_cast<int*>(ring_ptr + STAGES * C::STAGE_BYTES + 256);
    int* first = tiles + MAX_GROUPS + 1;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
    auto accum_full = [&](int a) { return bars + 8u * (2 * STAGES + a); };
    auto accum_empty = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * STAGES + 4);

    const int warp = __shfl_sync(~0u, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }      // full: weight copies, row copies
        for (int a = 0; a < 2; ++a) { mbar_init(accum_full(a), 1); mbar_init(accum_empty(a), EPI_WARPS * CTAS); }
        mbar_init(drain_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0 && elect_one()) { prefetch_map(map_x16); prefetch_map(map_x64); if (CTAS == 2) { prefetch_map(map_x8); prefetch_map(map_w); prefetch_map(map_sf); } }
    if (warp == 1) tc_alloc<CTAS>(smem_u32(tmem_slot), 512);
    tc_fence_before();
    build_table(p.rows, tiles, first);
    if (CTAS > 1) cluster_barrier();                                // both CTAs' barriers and tensor memory exist
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, *tmem_slot, 0);

    const int KT = (p.K + C::K_STEP - 1) / C::K_STEP, KT128 = (p.K + 127) / 128;
    const int ftiles = (p.N + C::FEATURES - 1) / C::FEATURES;
    Walk walk(tiles, first, p.rows.groups, ftiles);

    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1u) : 0, u_begin = blockIdx.x / CTAS, u_step = gridDim.x / CTAS;
    // The kernel before this one quantises the rows.  It lets this one start when everything before it has completed, so that
    // all but its own output may be read at once: the weights are on their way while the rows are quantised.
    // (The kernel behind this one may come up too; it waits for this one's end before it touches memory.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0 || warp == 3) {
        // ---------------- copies: weights and their scales (warp 0), rows (warp 3) ----------------
        bool ok = true;
        RingAt<STAGES> at;
        uint32_t issued = 0;
        for (int u = u_begin; u < walk.total && ok; u += u_step) {
            const Unit t = walk.at(u, C::FEATURES);
            const uint32_t n = uniform(t.padded()), mine = n / CTAS;                             // rows that this CTA brings
            const int row = uniform(t.row) + rank * (int)mine;
            // (features in tiles of 128; the second CTA of a pair whose first one has the last of them reads that again and stores nothing)
            const int ftile = min(uniform(t.ftile) * CTAS + rank, (p.N + 127) / 128 - 1);
            const uint8_t* w = p.w + (size_t)uniform(t.g) * p.w_group + (size_t)ftile * KT * C::Tile::BYTES;
            const uint8_t* x_sf = p.x_sf + (size_t)uniform(t.begin / p.rows.width + t.g + t.tile) * KT128 * (C::X_CHUNKS * 512);
            const uint32_t x_chunks = n > 128 ? 2 : 1;
            const int w_line = (int)((w - p.w) >> 7), sf_line = (int)((x_sf - p.x_sf) >> 7);     // a pair's maps are of lines of 128 bytes
            for (int kt = 0; kt < KT; ++kt, ++issued, at.step()) {
                ok = mbar_wait(empty_bar(at.s), at.phase ^ 1u, p.status, ST_PRODUCER_TIMEOUT);      // (a fresh barrier's phase before counts as complete)
                if (!ok) break;
                const uint32_t st = ring + at.s * C::STAGE_BYTES, full = full_bar(at.s);
                if (elect_one()) {
                    if (CTAS == 2) {
                        // both CTAs' copies complete the leader's barrier, where both CTAs' bytes are expected
                        const uint32_t both = map_to_rank(full, 0);
                        if (warp == 0) {
                            if (rank == 0) mbar_expect_tx(full, 2u * C::Tile::BYTES);
                            tma_load_2d_pair(st, &map_w, 0, w_line + kt * (C::Tile::BYTES / 128), both);
                        } else {
                            if (rank == 0) mbar_expect_tx(full, 2u * (mine * 128u + C::SF_STEPS * C::X_CHUNKS * 512u));
                            uint32_t r = 0;
                            for (; r + 64 <= mine; r += 64) tma_load_2d_pair(st + C::X + r * 128, &map_x64, kt * C::K_STEP, row + r, both);
                            for (; r + 16 <= mine; r += 16) tma_load_2d_pair(st + C::X + r * 128, &map_x16, kt * C::K_STEP, row + r, both);
                            if (r < mine) tma_load_2d_pair(st + C::X + r * 128, &map_x8, kt * C::K_STEP, row + r, both);
                            tma_load_2d_pair(st + C::SFX, &map_sf, 0, sf_line + kt * (C::SF_STEPS * C::X_CHUNKS * 4), both);
                        }
                    } else if (warp == 0) {
                        const uint8_t* block = w + (size_t)kt * C::Tile::BYTES;
                        mbar_expect_tx(full, C::Tile::BYTES);
                        bulk_load(st, block, C::Tile::CODES, full);
                        bulk_load(st + C::SFW, block + C::Tile::CODES, C::SF_STEPS * 512, full);
                    } else {
                        mbar_expect_tx(full, mine * 128u + C::SF_STEPS * x_chunks * 512u);
                        uint32_t r = 0;
                        for (; r + 64 <= mine; r += 64) tma_load_2d(st + C::X + r * 128, &map_x64, kt * C::K_STEP, row + r, full);
                        for (; r + 16 <= mine; r += 16) tma_load_2d(st + C::X + r * 128, &map_x16, kt * C::K_STEP, row + r, full);
#pragma unroll
                        for (int c = 0; c < C::SF_STEPS; ++c)
                            bulk_load(st + C::SFX + c * C::X_CHUNKS * 512, x_sf + (size_t)(kt * C::SF_STEPS + c) * (C::X_CHUNKS * 512),
                                      x_chunks * 512u, full);
                    }
                }
                __syncwarp();
            }
        }
        // Every copy this warp started must have landed before the CTA gives its shared memory back (returns at once in a run that went
        // well): the stage is full, or, where the leader's barrier tells that, the products have read it.
        for (uint32_t j = issued > (uint32_t)STAGES ? issued - STAGES : 0u; j < issued; ++j)
            mbar_wait(rank == 0 ? full_bar(j % STAGES) : empty_bar(j % STAGES), (j / STAGES) & 1, p.status, ST_PRODUCER_TIMEOUT);
    } else if (warp == 1 && rank == 1) {
        // the leader issues the products of both
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        // One thread's issue rate is what a narrow tile's products run at, so everything here is uniform over the warp (the
        // instructions take their operands from uniform registers) and the thread is elected.  The scales of a stage are copied
        // to tensor memory before the products of the stage in front of it, into the other set of columns: right in front of their own
        // products the copies hold up the tensor pipe (256 x 240 x 128: 1330 -> 1060 cycles).
        uint32_t count = 0, set = 0;
        bool ok = true, copied = false;
        RingAt<STAGES> at;
        int u = u_begin;
        Unit next = u < walk.total ? walk.at(u, C::FEATURES) : Unit{};
        // of a pair: what the other CTA's copies completed and its epilogue arrived at
        auto wait = [&](uint32_t bar, uint32_t parity) {
            return CTAS == 1 ? mbar_wait(bar, parity, p.status, ST_MMA_TIMEOUT) : mbar_wait_cluster(bar, parity, p.status, ST_MMA_TIMEOUT);
        };
        auto copy_scales = [&](int s, uint32_t into, uint32_t n) {
            const uint32_t from = ring + s * C::STAGE_BYTES, sfw = tmem + C::SFW_COL + into, sfx = tmem + C::SFX_COL + into;
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < C::SF_STEPS; ++c) {
                    const uint32_t w = from + C::SFW + c * 512, x = from + C::SFX + c * C::X_CHUNKS * 512;
                    tc_copy_scales<CTAS>(sfw + 8 * c, smem_desc(w, 0, 128, LAYOUT_NONE));
                    tc_copy_scales<CTAS>(sfx + 8 * c, smem_desc(x, 0, 128, LAYOUT_NONE));
                    if (C::X_CHUNKS == 2 && n > 128) tc_copy_scales<CTAS>(sfx + 8 * c + 4, smem_desc(x + 512, 0, 128, LAYOUT_NONE));
                }
            }
            __syncwarp();
        };
        for (; u < walk.total && ok; u += u_step, ++count) {
            const uint32_t n = uniform(next.padded());
            const bool more = u + u_step < walk.total;
            if (more) next = walk.at(u + u_step, C::FEATURES);
            const uint32_t next_n = uniform(next.padded());
            const uint32_t idesc = p.idesc | ((n >> 3) << 17);
            const int buf = (int)(count & 1u);
            // the first product into an accumulator overwrites it: the epilogue must have read what it held
            if (count >= 2) ok = wait(accum_empty(buf), ((count >> 1) - 1) & 1);
            tc_fence_after();
            const uint32_t d = tmem + buf * C::ACC_STRIDE;
            for (int kt = 0; kt < KT && ok; ++kt, set ^= C::SF_COLS) {
                const uint32_t st = ring + at.s * C::STAGE_BYTES, empty = empty_bar(at.s);
                if (!copied) {
                    ok = wait(full_bar(at.s), at.phase);
                    tc_fence_after();
                    if (!ok) break;
                    copy_scales(at.s, set, n);
                }
                copied = false;
                at.step();
                if ((kt + 1 < KT || more) && (CTAS == 1 ? mbar_test_wait(full_bar(at.s), at.phase) : mbar_test_wait_cluster(full_bar(at.s), at.phase))) {
                    tc_fence_after();
                    copy_scales(at.s, set ^ C::SF_COLS, kt + 1 < KT ? n : next_n);
                    copied = true;
                }
                const uint64_t w_desc = smem_desc(st, 16, 1024, LAYOUT_SW128), x_desc = smem_desc(st + C::X, 16, 1024, LAYOUT_SW128);
                const uint32_t sfw = tmem + C::SFW_COL + set, sfx = tmem + C::SFX_COL + set;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t acc = (kt > 0 || k > 0) ? 1u : 0u;
                        // scale byte k of a column; 64 elements of 4-bit pairs: bytes (0, 1) or (2, 3) of step k / 2
                        const uint32_t id = C::MXF4 ? (k & 1u) * 2u : k, step = C::MXF4 ? 8 * (k >> 1) : 0u;
                        tc_mma<CTAS, C::MXF4>(d, w_desc + 2 * k, x_desc + 2 * k, idesc | (id << 29) | (id << 4), sfw + step, sfx + step, acc);
                    }
                    tc_commit<CTAS>(empty);                                             // frees the stage once these products have read it
                }
                __syncwarp();
            }
            if (elect_one()) tc_commit<CTAS>(accum_full(buf));
            __syncwarp();
        }
        if (!ok) {
            // unwinding after a wait that ran out: the MMAs already issued must finish before tensor memory is freed
            if (elect_one()) tc_commit<CTAS>(drain_bar);
            __syncwarp();
            mbar_wait(drain_bar, 0, nullptr, 0);
        }
    } else if (warp >= FIRST_EPI_WARP) {
        // ---------------- epilogue ----------------
        // A warp takes 16 rows x 32 features at a time: tensor memory (a feature per lane) -> its own 2 KiB of shared memory
        // -> four consecutive features per lane, 8 lanes a row: loads of the second operand and stores are whole 64-byte
        // (fp32: 128-byte) segments.  The second operand of the next 16 rows is requested before the current ones are worked on, that of a
        // tile's first ones before the accumulator is complete.
        typedef typename Elem<DT>::T T;
        const int q = warp & 3, side = (warp - FIRST_EPI_WARP) >> 2;      // lane quadrant; the warps of one take 16-row chunks in turn
        const int er = lane >> 3, ef = q * 32 + (lane & 7) * 4;           // this lane's row (of every four) and first feature
        float* slot = reinterpret_cast<float*>(ring_ptr + STAGES * C::STAGE_BYTES + C::TABLE_END) + (warp - FIRST_EPI_WARP) * 512;
        T* out = reinterpret_cast<T*>(p.out);
        const T* extra = reinterpret_cast<const T*>(p.extra);
        bool ok = true;
        uint32_t count = 0;
        for (int u = u_begin; u < walk.total && ok; u += u_step, ++count) {
            const Unit t = walk.at(u, C::FEATURES);
            const int buf = (int)(count & 1u), f0 = t.f0 + rank * 128, f = f0 + ef;
            const int chunks = (t.rows + 15) >> 4;
            Four<T> e[4];
            auto request = [&](int c) {
                if (p.extra_mode == X_NONE) return;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = c * 16 + i * 4 + er;
                    if (r < t.rows) load_four(extra + (size_t)(t.row + r) * p.N + f, p.N - f, p.vector, e[i]);
                }
            };
            if (p.extra_mode != X_NONE && f0 < p.N) {
                // the whole tile of the second operand on its way to L2 while the products are formed: 128-byte lines, rows dealt to the threads
                const int bytes = min(128, p.N - f0) * (int)sizeof(T), lines = (bytes + 127) >> 7;
                for (int i = threadIdx.x - FIRST_EPI_WARP * 32; i < t.rows * lines; i += EPI_WARPS * 32)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(extra + (size_t)(t.row + i / lines) * p.N + f0) +
                                                                  min(i % lines * 128, bytes - 1)));
            }
            float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (p.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < 4; ++i) if (f + i < p.N) bias[i] = widen(reinterpret_cast<const T*>(p.bias)[(size_t)t.g * p.N + f + i]);
            }
            if (side < chunks) request(side);
            ok = mbar_wait(accum_full(buf), (count >> 1) & 1, p.status, ST_EPILOGUE_TIMEOUT);
            tc_fence_after();
            if (!ok) break;
            for (int c = side; c < chunks; c += EPI_SIDES) {
                uint32_t r[32];
                tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + buf * C::ACC_STRIDE + c * 16, r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < 16; ++j) slot[j * 32 + lane] = __uint_as_float(r[j]);
                __syncwarp();
                Four<T> now[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) now[i].w = e[i].w;
                if (c + EPI_SIDES < chunks) request(c + EPI_SIDES);
                T* at = out + (size_t)(t.row + c * 16 + er) * p.N + f;
                const int rows = (t.rows - c * 16 - er + 3) >> 2, left = p.N - f;
                finish_any(p.act, slot, lane, bias, now, p.extra_mode, at, p.N, rows, left, p.vector);
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { if (rank == 0) mbar_arrive(accum_empty(buf)); else arrive_after_tensor_reads(accum_empty(buf), 0); }
        }
        if (p.zero_rest) zero_rows_outside(out, first[0], first[p.rows.groups], p.rows.rows, p.N, threadIdx.x - FIRST_EPI_WARP * 32, EPI_WARPS * 32);
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS > 1) cluster_barrier();                                // neither CTA leaves while the other reads its memory or arrives on its barriers
    if (warp == 1) {
        tc_fence_after();
        tc_dealloc<CTAS>(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------------
// rows: reference codes + scales -> hardware codes and scale words
// ------------------------------------------------------------------------------------------------
struct CodeTables {
    uint8_t plain[256];     // reference code -> hardware code of the same value
    uint8_t halved[256];    // reference code -> hardware code of half the value, half to even
    uint32_t bad[8];        // bit c: reference code c is one that the hardware reads as Inf / NaN
};

// One thread per feature and 32-element block of a group (blockIdx.y), those that only fill up the last tile and step included
// (codes 0, scale 2^0).
__global__ void __launch_bounds__(256) pack_weights_kernel(const uint8_t* __restrict__ scales, const uint8_t* __restrict__ elements, int64_t N, int64_t K,
                                                           int nibbles, uint8_t* __restrict__ packed, const __grid_constant__ CodeTables t) {
    __shared__ uint8_t s_plain[256], s_halved[256];
    s_plain[threadIdx.x] = t.plain[threadIdx.x];
    s_halved[threadIdx.x] = t.halved[threadIdx.x];
    __syncthreads();
    const int blocks_per_step = nibbles ? 8 : 4, tile_bytes = nibbles ? WeightTile<true>::BYTES : WeightTile<false>::BYTES;
    const int64_t steps = nibbles ? WeightTile<true>::steps(K) : WeightTile<false>::steps(K), blocks = steps * blocks_per_step, features = (N + 127) / 128 * 128;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= features * blocks) return;
    const int64_t f = i / blocks, kb = i - f * blocks;
    const int r = (int)(f % 128), b = (int)(kb % blocks_per_step);
    uint8_t* tile = packed + (blockIdx.y * (features / 128 * steps) + f / 128 * steps + kb / blocks_per_step) * tile_bytes;
    uint4 c[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    uint32_t scale = 127u;
    if (f < N && kb * 32 < K) {
        const int64_t block = ((int64_t)blockIdx.y * N + f) * (K / 32) + kb;
        const uint4* from = reinterpret_cast<const uint4*>(elements + block * 32);
        c[0] = from[0];
        c[1] = from[1];
        scale = scales[block];
    }
    const uint8_t* cb = reinterpret_cast<const uint8_t*>(c);
    uint8_t* row = tile + r * 128;
    if (nibbles) {
        uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j >> 3] |= (uint32_t)(cb[j] & 0xFu) << (4 * (j & 7));
        *reinterpret_cast<uint4*>(row + ((b ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
        bool any_bad = false;
#pragma unroll
        for (int j = 0; j < 32; ++j) any_bad |= (t.bad[cb[j] >> 5] >> (cb[j] & 31)) & 1u;
        const uint8_t* lut = any_bad ? s_halved : s_plain;
        uint4 o[2];
        uint8_t* ob = reinterpret_cast<uint8_t*>(o);
#pragma unroll
        for (int j = 0; j < 32; ++j) ob[j] = lut[cb[j]];
        *reinterpret_cast<uint4*>(row + (((2 * b) ^ (r & 7)) << 4)) = o[0];
        *reinterpret_cast<uint4*>(row + (((2 * b + 1) ^ (r & 7)) << 4)) = o[1];
        if (any_bad && scale < 255u) ++scale;
    }
    tile[WeightTile<false>::CODES + (b >> 2) * 512 + (r % 32) * 16 + (r / 32) * 4 + (b & 3)] = (uint8_t)scale;
}

// Operand of the product: codes, scale chunks, chunks per 128-element step.
struct RowOperand {
    uint8_t *codes, *sf;
    int K, chunks, nibbles;
};

// One thread per row and 32-element block, padding blocks of the last 128 elements included (scale 2^0; the copies fill their
// codes with zeros).  A row index outside x gives a row of zeros.
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint8_t* __restrict__ scales, const uint8_t* __restrict__ elements,
                                                        const void* __restrict__ row_index, int index64, int64_t rows_in, const Groups g,
                                                        const RowOperand o_, const __grid_constant__ CodeTables t) {
    __shared__ uint8_t s_plain[256], s_halved[256];
    __shared__ int s_tiles[MAX_GROUPS + 1], s_first[MAX_GROUPS + 1];
    s_plain[threadIdx.x] = t.plain[threadIdx.x];
    s_halved[threadIdx.x] = t.halved[threadIdx.x];
    build_table(g, s_tiles, s_first);
    const int K = o_.K, blocks = (K + 127) / 128 * 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)g.rows * blocks) return;
    const int row = (int)(i / blocks), kb = (int)(i - (int64_t)row * blocks);
    if (row < s_first[0] || row >= s_first[g.groups]) return;
    int lo = 0, hi = g.groups;                           // the last group that begins at or before the row
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_first[mid] <= row) lo = mid; else hi = mid; }
    uint8_t* codes = o_.codes;
    uint8_t* sf_at = o_.sf + Place(g, lo, s_first[lo], s_first[lo + 1], row).at(kb, (K + 127) / 128, o_.chunks);
    if (kb * 32 >= K) { *sf_at = 127; return; }
    int64_t src = row;
    if (row_index != nullptr)
        src = index64 ? reinterpret_cast<const long long*>(row_index)[row] : (int64_t)reinterpret_cast<const int*>(row_index)[row];
    uint4 c[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    uint32_t scale = 127u;
    if (src >= 0 && src < rows_in) {
        const uint4* from = reinterpret_cast<const uint4*>(elements + src * K + kb * 32);
        c[0] = from[0];
        c[1] = from[1];
        scale = scales[src * (K / 32) + kb];
    }
    const uint8_t* cb = reinterpret_cast<const uint8_t*>(c);
    if (o_.nibbles) {
        uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j >> 3] |= (uint32_t)(cb[j] & 0xFu) << (4 * (j & 7));
        *reinterpret_cast<uint4*>(codes + (int64_t)row * (K / 2) + kb * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        *sf_at = (uint8_t)scale;
        return;
    }
    bool any_bad = false;
#pragma unroll
    for (int j = 0; j < 32; ++j) any_bad |= (t.bad[cb[j] >> 5] >> (cb[j] & 31)) & 1u;
    const uint8_t* lut = any_bad ? s_halved : s_plain;
    uint4 o[2];
    uint8_t* ob = reinterpret_cast<uint8_t*>(o);
#pragma unroll
    for (int j = 0; j < 32; ++j) ob[j] = lut[cb[j]];
    uint4* to = reinterpret_cast<uint4*>(codes + (int64_t)row * K + kb * 32);
    to[0] = o[0];
    to[1] = o[1];
    *sf_at = (uint8_t)((any_bad && scale < 255u) ? scale + 1u : scale);
}

// One pass from x to the operand (built-in round-to-nearest formats, 16-byte aligned rows).  One CTA per row segment: the row's group and
// place are looked up once.  A lane has four accesses of 8 elements; of the four lanes of a block, lane i derives the header of
// access i and stores its scale.  Bound by memory (x read once, gathered rows mostly from L2) and integer issue about equally:
// 8192 gathered rows of 2048 to E2M1 in 21 us, cold.  Several rows per CTA with the group looked up by each warp alone: 1 us slower at
// 192 and at 8192 rows.
constexpr int QUANT_ACCESSES = 4;                // accesses of 8 elements per lane = lanes of a block
template <class KIn, class F, int OUT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* x, const void* row_index, int index64, int64_t rows_in, const Groups g,
                                                            const RowOperand o_, int segments, int early) {
    __shared__ int s_two[2];
    // everything before this kernel has completed; then the product may start: until it waits for this kernel it only reads what is older
    // (what an earlier kernel may still be writing when this one starts is not loaded as read-only data: such loads could move in front)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int BYTES = 8 * KIn::size;
    const int K = o_.K;
    const int row = (int)(blockIdx.x / (unsigned)segments);
    const int first = ((int)(blockIdx.x % (unsigned)segments) * QUANT_ACCESSES * (int)blockDim.x + (int)threadIdx.x) * 8;
    int64_t src = row;
    if (row_index != nullptr)
        src = index64 ? reinterpret_cast<const long long*>(row_index)[row] : (int64_t)reinterpret_cast<const int*>(row_index)[row];
    const bool there = src >= 0 && src < rows_in;                            // a row index outside x gives a row of zeros
    const char* from = reinterpret_cast<const char*>(x) + src * K * KIn::size;
    const uint32_t fill = there ? one_bits<KIn>() : 0u;                       // lanes behind K do not hold up the others' short form
    uint32_t raw[QUANT_ACCESSES][BYTES / 4];
#pragma unroll
    for (int a = 0; a < QUANT_ACCESSES; ++a) {
        const int k = first + a * (int)blockDim.x * 8;
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = there && k < K ? __ldcg(reinterpret_cast<const uint4*>(from + (int64_t)k * KIn::size) + i) : make_uint4(fill, fill, fill, fill);
            raw[a][4 * i] = v.x; raw[a][4 * i + 1] = v.y; raw[a][4 * i + 2] = v.z; raw[a][4 * i + 3] = v.w;
        }
    }
    const Place place = find_row(g, row, s_two);
    if (place.slot < 0) return;
    const int lane = threadIdx.x & 31, sub = lane & 3;
    uint32_t hi[QUANT_ACCESSES], lo[QUANT_ACCESSES];
#pragma unroll
    for (int a = 0; a < QUANT_ACCESSES; ++a) {
        part_range<KIn, 8>(raw[a], hi[a], lo[a]);
        hi[a] = part_reduce<KIn, 8>(hi[a]);
    }
    uint32_t mine = hi[0];
#pragma unroll
    for (int a = 1; a < QUANT_ACCESSES; ++a) mine = sub == a ? hi[a] : mine;
    const uint2 header = part_header<KIn, F>(mine);
    uint32_t scale = 0u;
#pragma unroll
    for (int a = 0; a < QUANT_ACCESSES; ++a) {
        const int k = first + a * (int)blockDim.x * 8, from_lane = (lane & ~3) + a;
        uint32_t o[OUT == 5 ? 1 : 2];
        const uint2 of_block = make_uint2(__shfl_sync(~0u, header.x, from_lane), __shfl_sync(~0u, header.y, from_lane));
        const uint32_t sbyte = part_encode<KIn, F, OUT, 8>(raw[a], lo[a], of_block, o);
        scale = sub == a ? sbyte : scale;
        if (k < K) {
            if constexpr (OUT == 5) *reinterpret_cast<uint32_t*>(o_.codes + ((int64_t)row * K + k) / 2) = o[0];
            else *reinterpret_cast<uint2*>(o_.codes + (int64_t)row * K + k) = make_uint2(o[0], o[1]);
        }
    }
    const int kb = (first + sub * (int)blockDim.x * 8) >> 5;                     // the block of access `sub`
    if (kb * 32 < K) {
        uint8_t* at = o_.sf + place.at(kb, (K + 127) / 128, o_.chunks);
        *at = (uint8_t)scale;
        if (kb * 32 + 32 == K) for (int i = 1; i < 4 - (kb & 3); ++i) at[i] = 127;     // K blocks that only fill up the last 128 elements
    }
    if (!early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// MXQ_ESIZE: not covered (a rounding mode other than to nearest, unaligned rows), take extract + pack_rows_kernel
static int quantize_rows(const void* x, int x_dtype, const void* row_index, int index64, int64_t rows_in, const Groups& g, int eb, int fb, int rm,
                         const RowOperand& o, cudaStream_t st) {
    const int64_t K = o.K, rows = g.rows;
    const int64_t lanes = (K / 8 + QUANT_ACCESSES - 1) / QUANT_ACCESSES;
    const int block = lanes >= 256 ? 256 : (int)((lanes + 31) / 32 * 32);
    const int64_t segments = (K / 8 + (int64_t)block * QUANT_ACCESSES - 1) / ((int64_t)block * QUANT_ACCESSES);
    if (rm != MXQ_RN || reinterpret_cast<uintptr_t>(x) % 16 != 0 || rows * segments > (1ll << 31) - 1) return MXQ_ESIZE;
    // a short grid lets the product's CTAs come up beside it (777 rows: 15.1 -> 14.4 us the call); a long one keeps the SMs' registers to itself until its end
    const int early = rows * segments <= 32 * sm_count();
    int rc = MXQ_ESIZE;
    with_kind(x_dtype, [&](auto kin) {
        using KIn = decltype(kin);
        with_row_format(eb, fb, o.nibbles, [&](auto fmt, auto out) {
            rc = launch_after(quantize_rows_kernel<KIn, decltype(fmt), decltype(out)::value>, (unsigned)(rows * segments), (unsigned)block, 0, 1, st, x, row_index,
                              index64, rows_in, g, o, (int)segments, early);
        });
    });
    return rc;
}

// slots of the rows' scales, one per row tile
static int64_t tile_slots(int64_t rows, int64_t groups, int64_t width) { return rows / width + groups + 1; }

template <class C, int DT>
static int launch(const Params& p, const uint8_t* x_codes, cudaStream_t st) {
    static bool attr_done[MAX_DEVICES] = {false};
    const cudaError_t e = raise_smem_limit(grouped_kernel<C, DT>, C::SMEM_BYTES, attr_done);
    if (e != cudaSuccess) { set_last_cuda_error(e); return MXQ_ELAUNCH; }
    CUtensorMap mx64, mx16, mx8, mw, msf;
    const Groups& g = p.rows;
    if (!make_map(&mx64, x_codes, g.rows, p.K, 64, C::MXF4) || !make_map(&mx16, x_codes, g.rows, p.K, 16, C::MXF4) ||
        (C::CTAS == 2 && !make_map(&mx8, x_codes, g.rows, p.K, 8, C::MXF4))) return MXQ_ELAUNCH;
    if constexpr (C::CTAS == 2) {
        // a block of the weights, a stage's scales of the rows, as lines of 128 bytes
        const int64_t sf_lines = tile_slots(g.rows, g.groups, g.width) * ((p.K + 127) / 128) * (C::X_CHUNKS * 4);
        if (!make_line_map(&mw, p.w, g.groups * (p.w_group / 128), C::Tile::BYTES / 128) || !make_line_map(&msf, p.x_sf, sf_lines, C::SF_STEPS * C::X_CHUNKS * 4))
            return MXQ_ELAUNCH;
    } else {
        mx8 = mw = msf = mx16;                                       // a pair's only
    }
    const int64_t units = most_units(g, p.N, C::FEATURES);
    const int64_t room = sm_count() / C::CTAS;
    return launch_after(grouped_kernel<C, DT>, (unsigned)((units < room ? units : room) * C::CTAS), C::THREADS, C::SMEM_BYTES, C::CTAS, st, mx64, mx16, mx8, mw, msf, p);
}

template <class C>
static int launch_dt(const Params& p, int dt, const uint8_t* x_codes, cudaStream_t st) {
    if (dt == MXQ_F32) return launch<C, MXQ_F32>(p, x_codes, st);
    if (dt == MXQ_BF16) return launch<C, MXQ_BF16>(p, x_codes, st);
    return launch<C, MXQ_F16>(p, x_codes, st);
}

// element formats of the tensor-core path
static bool valid_mx_preset(int eb, int fb) {
    return (eb == 4 && fb == 3) || (eb == 5 && fb == 2) || (eb == 2 && (fb == 3 || fb == 1)) || (eb == 3 && fb == 2);
}
static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Kernel and tile width of a call, from the sizes that the host knows.
enum Shape { DECODE, NARROW, TALL, PAIR };
struct Plan {
    Shape shape;                 // the kernel for few rows, where x and its format allow; tiles of up to 128 rows; up to 240 (224 of E2M1 pairs); these on a pair of CTAs
    int width;                   // rows per tile at most
    int chunks() const { return shape <= NARROW ? 1 : 2; }
    int64_t sf_bytes(int64_t rows, int64_t groups, int64_t K) const { return tile_slots(rows, groups, width) * ((K + 127) / 128) * chunks() * 512; }
};
// Whether the kernel for few rows is the faster one.  There every CTA quantises the rows for its own features, some 62 ns a row and 128
// elements (`load`: that on every SM), which from some 8 rows on takes longer than the weights' copies; a group's tiles of 16 rows each
// read its weights.  Narrow tiles have a second launch in front (calls from the host: 14.5 us against 9.5, while the GPU takes less), and no split
// of K: they need N to fill the SMs.  Measured with cold weights, microseconds, few rows / narrow tiles:
//   linear, 4096 -> 14336: 15.0 / 15.4 (6 rows), 16.0 / 15.4 (8), 18.5 / 15.4 (10), 31.6 / 15.4 (16); 8192 -> 28672: 40.5 / 45.9 (8), 50.8 / 45.9 (10);
//     14336 -> 4096: 28.6 / 33.1 (16); 4096 -> 4096: 13.3 / 13.4 (16);
//   4-bit pairs, 4096 -> 14336: 10.4 / 10.9 (4), 11.7 / 10.9 (6); 8192 -> 28672: 26.7 / 27.8 (6), 31.9 / 27.8 (8); 14336 -> 4096: 18.9 / 20.8 (12), 21.4 / 20.8 (14);
//   64 experts, 2048 -> 1024, rows dealt evenly: 26.1 / 29.4 (2 a group), 26.7 / 29.8 (4); by uneven popularity: 25.4 / 23.5 (2), 28.8 / 28.9 (3),
//     35.4 / 29.6 (4), 39.3 / 31.4 (8); 8 experts, 4096 -> 14336, uneven: 65.4 / 71.1 (2), 69.4 / 71.2 (3), 76.3 / 71.3 (4).  (The host knows the average only.)
//   small ones, called from the host: linear, 1024 -> 14336: 11.7 / 14.4 (16 rows, load 6 us); 2048 -> 12288: 12.0 / 14.5 (12, 7.7 us), 17.9 / 14.5 (16, 10.3 us);
//     uneven experts: 16 of 1024 -> 1024: 10.0 / 14.8 (3 a group, 1.3 us); 4 of 4096 -> 2048: 11.3 / 14.6 (3, 2.6 us), 17.8 / 14.6 (4, 3.4 us).
static bool takes_few(int64_t rows, int64_t groups, int64_t N, int64_t K, bool fp4, int64_t sms) {
    const int64_t ftiles = (N + 127) / 128;
    const double load = (double)rows * (double)((K + 127) / 128) * (double)ftiles * 0.062 / (double)sms;          // microseconds
    if (groups > 1) return rows <= 2 * groups || (rows / groups <= decode_rows() / 2 && load <= 2.5);
    const bool fills = ftiles * 2 > sms;
    return rows <= (load <= 8.0 ? decode_rows() : fp4 ? (fills ? 5 : 12) : fills ? decode_rows() / 2 : decode_rows());
}
// The tiles that take the fewest estimated nanoseconds of the whole GPU: rounds of tiles x steps of K x what a step takes.  That is
// what one thread issues (215) at least; else, for one CTA, what L2 gives all SMs together (13.4 TB/s measured: 47.6 KB of a 240-row step in
// 534 ns on 148 SMs, 33.3 KB of a 128-row step in 364), for a pair the products and a fixed part (347 at 128 rows, 483 at 224; under the power
// cap, which large products run into).  Measured, microseconds, one CTA / pair: 8192 rows, 14336 x 4096: 570 / 570 (128 rows), 525 / 477 (192),
// 482 / 458 (224); 192 rows, 4096 x 4096: 20.6 / 20.0 (64), 19.4 / 19.9 (128); 2048 rows, 2048 x 2048: 25.9 (128), 24.8 (240), 29.8 (pair, 240).
// (One CTA with 256 x 240 has the pair's bytes, but fills tensor memory: its epilogue overlaps nothing, 544.)
// The estimate ranks tiles of one problem and no more: it counts steps of K and no epilogue, with constants of 8-bit products, and lies below the
// kernel's time where K is short or operands have four bits.  Estimate / kernel alone, microseconds: 192 rows, 4096 x 4096: 6.9 / 17.7; 3001 rows
// over 17 experts, 520 x 1184: 2.6 / 17.2; 4-bit pairs, 4096 x 4096 x 4096: 34 / 41, 8192 rows over 32 experts, 2048 x 2048: 19 / 48.
static Plan make_plan(int64_t rows, int64_t groups, int64_t N, int64_t K, bool fp4, int64_t sms) {
    if (takes_few(rows, groups, N, K, fp4, sms)) return Plan{DECODE, Narrow::BT};
    const int64_t each = (rows + groups - 1) / groups, ftiles = (N + 127) / 128, steps = (K + (fp4 ? 255 : 127)) / (fp4 ? 256 : 128);
    Plan best{NARROW, 0};
    double least = 0.0;
    for (int ctas = 1; ctas <= 2; ++ctas)
        for (int width = ctas == 1 ? 48 : 160; width <= (fp4 ? TallFp4::BT : Tall::BT); width += 16) {
            const int64_t per_group = (each + width - 1) / width, units = per_group * groups * ((ftiles + ctas - 1) / ctas), places = sms / ctas;
            if (ctas == 2 && units < 4 * places) continue;                // a few rounds: the coarser tiles' last one costs more than they save
            const double used = (double)(((each + per_group - 1) / per_group + 15) / 16 * 16), busy = units < places ? (double)units / places : 1.0;
            const double step = ctas == 1 ? (17.0 + 0.128 * used) * 11.05 * busy : 160.0 + 1.4 * used;
            const double cost = (double)((units + places - 1) / places * steps) * (step > 215.0 ? step : 215.0);
            if (best.width == 0 || cost < 0.98 * least) { best = Plan{ctas == 2 ? PAIR : width <= Narrow::BT ? NARROW : TALL, width}; least = cost; }
        }
    return best;
}

}  // namespace grouped
}  // namespace mxq

using namespace mxq;

extern "C" int mxq_mx_max_groups(void) { return grouped::MAX_GROUPS; }

extern "C" int64_t mxq_mx_packed_experts_bytes(int64_t groups, int64_t N, int64_t K, int nibbles) {
    if (groups <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return MXQ_EINVAL;
    return groups * (nibbles ? grouped::WeightTile<true>::group_bytes(N, K) : grouped::WeightTile<false>::group_bytes(N, K));
}

extern "C" int mxq_mx_pack_experts(const uint8_t* scales, const uint8_t* elements, int64_t groups, int64_t N, int64_t K, int eb, int fb, int nibbles,
                                   uint8_t* packed, int* hw_format, void* stream) {
    if (groups <= 0 || N <= 0 || K <= 0 || K % 32 != 0 || !scales || !elements || !packed || !hw_format) return MXQ_EINVAL;
    if (groups > grouped::MAX_GROUPS || groups * N > (1ll << 31) - 1 || K > (1 << 30)) return MXQ_ESIZE;
    if ((reinterpret_cast<uintptr_t>(elements) | reinterpret_cast<uintptr_t>(packed)) % 16 != 0) return MXQ_EINVAL;
    if (nibbles && (eb != 2 || fb != 1 || K % 256 != 0)) return MXQ_ESIZE;
    grouped::CodeTables t;
    int fmt;
    if (!hw_code_tables(eb, fb, t.plain, t.halved, t.bad, &fmt)) return MXQ_EINVAL;
    const int64_t steps = nibbles ? grouped::WeightTile<true>::steps(K) * 8 : grouped::WeightTile<false>::steps(K) * 4;
    const int64_t threads = (N + 127) / 128 * 128 * steps;
    if ((threads + 255) / 256 > (1ll << 31) - 1) return MXQ_ESIZE;
    grouped::pack_weights_kernel<<<dim3((unsigned)((threads + 255) / 256), (unsigned)groups), 256, 0, (cudaStream_t)stream>>>(scales, elements, N, K, nibbles, packed, t);
    const int rc = check_launch();
    if (rc == MXQ_OK) *hw_format = nibbles ? 5 : fmt;
    return rc;
}

// the decode kernel quantises by itself: no operand in memory
static bool takes_decode(const grouped::Plan& plan, const void* x, int round_mode) {
    return plan.shape == grouped::DECODE && round_mode == MXQ_RN && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}

static int64_t scratch_of(const grouped::Plan& plan, const void* x, int round_mode, int64_t rows_in, int64_t rows, int64_t K, int64_t groups) {
    if (rows == 0 || takes_decode(plan, x, round_mode)) return 0;
    return grouped::align256(rows * K) + grouped::align256(plan.sf_bytes(rows, groups, K)) + grouped::align256(rows_in * K) + grouped::align256(rows_in * K / 32);
}

extern "C" int64_t mxq_mx_grouped_scratch_bytes(const void* x, int round_mode, int64_t rows_in, int64_t rows, int64_t K, int64_t groups, int64_t N) {
    if (rows_in < 0 || rows < 0 || groups <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return MXQ_EINVAL;
    const int64_t sms = tc::sm_count();
    // whichever way the weight is packed
    return std::max(scratch_of(grouped::make_plan(rows, groups, N, K, false, sms), x, round_mode, rows_in, rows, K, groups),
                    scratch_of(grouped::make_plan(rows, groups, N, K, true, sms), x, round_mode, rows_in, rows, K, groups));
}

extern "C" int mxq_mx_grouped_linear(const mxq_grouped_linear_args* args) {
    if (!args) return MXQ_EINVAL;
    const auto [x, row_index, w_packed, offsets, out, bias, extra, scratch, status, stream, rows_in, rows, K, groups, N, scratch_bytes, x_dtype, x_exp_bits, x_frac_bits,
                x_round_mode, index64, offsets64, w_hw_format, activation, extra_mode, zero_rest] = *args;
    if (rows < 0 || rows_in < 0 || groups <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return MXQ_EINVAL;
    if (x_dtype != MXQ_F32 && x_dtype != MXQ_BF16 && x_dtype != MXQ_F16) return MXQ_EINVAL;
    if (activation < MXQ_ACT_NONE || activation > MXQ_ACT_SILU || extra_mode < MXQ_EXTRA_NONE || extra_mode > MXQ_EXTRA_ADD) return MXQ_EINVAL;
    if (row_index == nullptr && rows != rows_in) return MXQ_EINVAL;
    if (offsets == nullptr && groups != 1) return MXQ_EINVAL;
    if (groups > grouped::MAX_GROUPS || rows > (1 << 30) || N > (1 << 30) || K > (1 << 30) || groups * N > (1ll << 31) - 1) return MXQ_ESIZE;
    if (rows * ((K + 127) / 128 * 4) > (1ll << 31) * 255 || rows_in > (1 << 30)) return MXQ_ESIZE;
    if (rows == 0) return MXQ_OK;
    if ((!x && rows_in > 0) || !w_packed || !out || (extra_mode != MXQ_EXTRA_NONE && !extra)) return MXQ_EINVAL;
    if (reinterpret_cast<uintptr_t>(w_packed) % 16 != 0 || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return MXQ_EINVAL;
    // both operands E2M1 and the weight kept as nibbles: the 4-bit kind
    const bool x_e2m1 = x_exp_bits == 2 && x_frac_bits == 1;
    const bool fp4 = w_hw_format == 5;
    if (fp4 && (!x_e2m1 || K % 256 != 0)) return MXQ_EINVAL;
    if (!fp4 && w_hw_format != 0 && w_hw_format != 1) return MXQ_EINVAL;
    if (!grouped::valid_mx_preset(x_exp_bits, x_frac_bits) || x_round_mode < MXQ_RN || x_round_mode > MXQ_RZ) return MXQ_EINVAL;
    const int x_fmt = x_exp_bits == 5 ? 1 : 0;

    const grouped::Plan plan = grouped::make_plan(rows, groups, N, K, fp4, tc::sm_count());
    const int64_t needed = scratch_of(plan, x, x_round_mode, rows_in, rows, K, groups);
    if (needed > 0 && !scratch) return MXQ_EINVAL;
    if (scratch_bytes < needed) return MXQ_ESIZE;
    grouped::Params p{};
    p.w = w_packed;
    p.w_group = fp4 ? grouped::WeightTile<true>::group_bytes(N, K) : grouped::WeightTile<false>::group_bytes(N, K);
    p.out = out; p.bias = bias; p.extra = extra;
    p.rows = grouped::Groups{offsets, offsets64, (int)rows, (int)groups, plan.width};
    p.N = (int)N; p.K = (int)K;
    const uintptr_t four = x_dtype == MXQ_F32 ? 16 : 8;
    p.vector = N % 4 == 0 && reinterpret_cast<uintptr_t>(out) % four == 0 && reinterpret_cast<uintptr_t>(extra) % four == 0;
    p.act = activation; p.extra_mode = extra_mode; p.zero_rest = zero_rest; p.status = status;
    // formats of left (weight) and right (rows) operand, K-major both, E8M0 scales, M >> 4; E2M1 is 1 in the 4-bit kind's encoding
    p.idesc = (fp4 ? (1u << 7) | (1u << 10) : ((uint32_t)w_hw_format << 7) | ((uint32_t)x_fmt << 10)) | (1u << 23) | ((uint32_t)(128 >> 4) << 24);
    cudaStream_t st = (cudaStream_t)stream;
    if (takes_decode(plan, x, x_round_mode)) {
        p.rows.width = grouped::decode_rows();
        return grouped::launch_decode(p, x_dtype, x, row_index, index64, rows_in, x_exp_bits, x_frac_bits, fp4, st);
    }

    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* sf = codes + grouped::align256(rows * K);
    uint8_t* ref_codes = sf + grouped::align256(plan.sf_bytes(rows, groups, K));
    uint8_t* ref_scales = ref_codes + grouped::align256(rows_in * K);
    p.x_sf = sf;
    const grouped::RowOperand operand{codes, sf, (int)K, plan.chunks(), fp4};
    int rc = grouped::quantize_rows(x, x_dtype, row_index, index64, rows_in, p.rows, x_exp_bits, x_frac_bits, x_round_mode, operand, st);
    if (rc == MXQ_ESIZE) {
        if (rows_in > 0) {
            rc = mxq_mxfp_extract(x, x_dtype, ref_scales, ref_codes, rows_in * K, 32, x_exp_bits, x_frac_bits, 1, x_round_mode, stream);
            if (rc != MXQ_OK) return rc;
        }
        grouped::CodeTables tables;
        int fmt;
        if (!hw_code_tables(x_exp_bits, x_frac_bits, tables.plain, tables.halved, tables.bad, &fmt)) return MXQ_EINVAL;
        const int64_t threads = rows * ((K + 127) / 128 * 4);
        grouped::pack_rows_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(ref_scales, ref_codes, row_index, index64, rows_in, p.rows, operand, tables);
        rc = check_launch();
    }
    if (rc != MXQ_OK) return rc;
    using namespace grouped;
    if (plan.shape == PAIR) {
        p.idesc += (uint32_t)(128 >> 4) << 24;           // 256 features per instruction
        return fp4 ? launch_dt<PairFp4>(p, x_dtype, codes, st) : launch_dt<Pair>(p, x_dtype, codes, st);
    }
    if (plan.shape == TALL) return fp4 ? launch_dt<TallFp4>(p, x_dtype, codes, st) : launch_dt<Tall>(p, x_dtype, codes, st);
    return fp4 ? launch_dt<NarrowFp4>(p, x_dtype, codes, st) : launch_dt<Narrow>(p, x_dtype, codes, st);
}
