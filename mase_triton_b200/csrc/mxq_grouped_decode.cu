// The grouped products for few rows (a decoding step): one kernel, in which the rows are quantised by the CTAs that multiply them.
//
// What bounds such a call is one read of the weights and, below some 20 us, everything in front of and behind it: launches, the
// ramp of the grid, a second kernel's hand-over.  So
//   * five warps of every CTA (four for 4-bit pairs) quantise the rows of its tile (16 at most) as they go along K, straight into the ring of
//     shared memory that the tensor cores read, a stage each in turn: one warp's way through a stage (a load, the block
//     maximum, the rounding, a proxy fence) takes far longer than the stage's products.  Every CTA repeats this for its own features,
//     out of L2 and beside the weights' copies, which take longer; there is no second launch, no operand in memory and no workspace;
//   * two CTAs fit on an SM (a ring of 95 KB each, 80 for 4-bit pairs; and for up to 1024 groups): one's start and end hide behind the other's copies, within a call and, with
//     the launch that may overlap the kernel before, between calls;
//   * where the features leave SMs idle, K is split over a cluster of 2 or 4 CTAs.  Each sums its part in tensor memory; the
//     partial sums go to the CTA that finishes those features through distributed shared memory and are added in the
//     order of the CTAs, so that results do not depend on which comes first.
// The layout of weights, the walk over the units and the epilogue are those of mxq_grouped.cu.
// Measured (replays in a row): 1 row, 4096 -> 14336, E4M3: 14.1 us (4.3 TB/s of all bytes; 9.3 at the copy rate); 2 rows over 8 such
// experts: 23.6 (5.1 TB/s); 5 rows, 14336 -> 4096, E3M2: 16.4.  256 rows over 64 experts, 2048 -> 1024 (which narrow tiles take by now, in 30.6): 32.4; there
// CTAs of one unit each in the hardware's order instead of CTAs that stay: 36.0; weights held back until the first rows have arrived, not
// just been asked for: 33.6.
#include "mxq_grouped.cuh"

namespace mxq {
namespace grouped {
namespace decode {

constexpr int ROWS = 16;                         // widest row tile: the narrowest the instruction takes
constexpr int FEATURES = 128;
constexpr int EPI_WARP = 4;
constexpr int THREADS = 352;                     // warps 0, 1: weight copies, MMA issuer; 4..7: epilogue; 2, 3, 8..10: quantisers
constexpr int X_BYTES = ROWS * 128;
constexpr int TMEM_COLS = 128;
constexpr int ACC_STRIDE = 32, SFW_COL = 64, SFX_COL = 96;

template <bool MXF4> struct Cfg {
    using Tile = WeightTile<MXF4>;
    static constexpr int K_STEP = Tile::K_STEP, SF_STEPS = Tile::SF_STEPS;
    static constexpr int STAGES = MXF4 ? 4 : 5;
    // a warp that took a stage more than one turn of the ring ahead would mistake the phase its barrier is in
    static constexpr int QUANT_WARPS = STAGES;
    static_assert(QUANT_WARPS <= STAGES && EPI_WARP + 2 + QUANT_WARPS <= THREADS / 32, "quantising warps");
    // a stage: row codes | a block of the weights, its scales behind its codes | scales of the rows, 512 bytes per 128 elements of K
    static constexpr int W = X_BYTES, SFW = W + Tile::CODES, SFX = W + Tile::BYTES;
    static constexpr int STAGE_BYTES = SFX + SF_STEPS * 512;
    static constexpr int SLOTS = 4 * 2048, EXCHANGE = 3 * 2048;                      // 32 features x 16 rows per epilogue warp, and per part received
    static constexpr int FIXED_BYTES = 1024 + STAGES * STAGE_BYTES + 256 + SLOTS;
    // behind these the group table and the exchange of a cluster; CTAs that share no unit have none
    static constexpr int smem_bytes(int groups, int split) { return FIXED_BYTES + (split > 1 ? EXCHANGE : 0) + 2 * (groups + 1) * 4; }
    static constexpr int per_sm(int groups, int split) { return 2 * (smem_bytes(groups, split) + 1024) <= 233472 ? 2 : 1; }
    static_assert(STAGE_BYTES % 1024 == 0, "the 128-byte swizzle repeats every 1024 bytes");
    static_assert(smem_bytes(MAX_GROUPS, 2) <= 232448, "more shared memory than a CTA can have");
    static_assert(per_sm(MAX_GROUPS, 1) == 2, "two CTAs fit on an SM");
};

struct Source {
    const void* x;
    const void* row_index;
    int index64;
    int64_t rows_in;
};

__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// DT: type of x, out, bias and extra; F, OUT: element format of the rows and what the tensor cores read of it
template <int DT, class F, int OUT>
__global__ void __launch_bounds__(THREADS, 2)
decode_kernel(const __grid_constant__ Params p, const __grid_constant__ Source src, int split) {
    constexpr bool MXF4 = OUT == 5;
    using C = Cfg<MXF4>;
    constexpr int STAGES = C::STAGES;
    typedef typename Elem<DT>::T T;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw);
    const uint32_t bars = ring + STAGES * C::STAGE_BYTES;            // full[S], empty[S], accum_full[2], accum_empty[2], drain, parts, rows requested, tmem slot
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring_ptr + STAGES * C::STAGE_BYTES + 8 * (2 * STAGES + 7));
    float* slots = reinterpret_cast<float*>(ring_ptr + STAGES * C::STAGE_BYTES + 256);
    int* tiles = reinterpret_cast<int*>(slots + C::SLOTS / 4);
    int* first = tiles + p.rows.groups + 1;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
    auto accum_full = [&](int a) { return bars + 8u * (2 * STAGES + a); };
    auto accum_empty = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
    const uint32_t drain_bar = bars + 8u * (2 * STAGES + 4), parts_bar = bars + 8u * (2 * STAGES + 5);
    const uint32_t rows_bar = bars + 8u * (2 * STAGES + 6);

    const int warp = __shfl_sync(~0u, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)(blockIdx.x % (unsigned)split) : 0;           // clusters are consecutive CTAs
    const int quads = 4 / split;                                                     // lane quadrants whose features a CTA finishes
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(accum_full(a), 1); mbar_init(accum_empty(a), 4); }
        mbar_init(drain_bar, 1);
        mbar_init(rows_bar, C::QUANT_WARPS);
        mbar_init(parts_bar, (split - 1) * quads + (split == 1 ? 1 : 0));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // What the kernels before this one write (rows, offsets, perhaps the weights) is read behind a wait for their end only: here
    // for offsets; without them every warp gets as far as its first access and waits there.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (p.rows.offsets != nullptr) dependency_wait();
    tc_fence_before();
    build_table(p.rows, tiles, first);
    if (split > 1) cluster_barrier();                                // every CTA's barriers exist before another one arrives there
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, *tmem_slot, 0);

    const int KT_all = (p.K + C::K_STEP - 1) / C::K_STEP;
    const int k_begin = rank * KT_all / split, KT = (rank + 1) * KT_all / split - k_begin;     // this CTA's steps of K, one at least
    const int ftiles = (p.N + FEATURES - 1) / FEATURES;
    const int u_begin = blockIdx.x / split, u_step = gridDim.x / split;
    Walk walk(tiles, first, p.rows.groups, ftiles);

    if (warp == 0) {
        // ---------------- weight copies ----------------
        bool ok = true;
        RingAt<STAGES> at;
        uint32_t issued = 0;
        for (int u = u_begin; u < walk.total && ok; u += u_step) {
            const Unit t = walk.at(u, FEATURES);
            const uint8_t* w = p.w + (size_t)uniform(t.g) * p.w_group + (size_t)uniform(t.ftile) * KT_all * C::Tile::BYTES;
            for (int kt = k_begin; kt < k_begin + KT; ++kt, ++issued, at.step()) {
                ok = mbar_wait(empty_bar(at.s), at.phase ^ 1u, p.status, ST_PRODUCER_TIMEOUT);      // (a fresh barrier's phase before counts as complete)
                if (!ok) break;
                const uint32_t st = ring + at.s * C::STAGE_BYTES, full = full_bar(at.s);
                // The weights that all CTAs ask for at once keep the memory busy for microseconds.  The first rows, which everything
                // waits for, are asked for in front of all but one stage of them.
                if (issued == 0) dependency_wait();
                if (issued == 1) mbar_wait(rows_bar, 0, p.status, ST_PRODUCER_TIMEOUT);
                if (elect_one()) {
                    mbar_expect_tx(full, C::Tile::BYTES);
                    bulk_load(st + C::W, w + (size_t)kt * C::Tile::BYTES, C::Tile::BYTES, full);
                }
                __syncwarp();
            }
        }
        // every copy must have landed before the CTA gives its shared memory back (returns at once in a run that went well)
        for (uint32_t j = issued > (uint32_t)STAGES ? issued - STAGES : 0u; j < issued; ++j)
            mbar_wait(full_bar(j % STAGES), (j / STAGES) & 1, p.status, ST_PRODUCER_TIMEOUT);
    } else if (warp == 1) {
        // ---------------- MMA issuer: uniform over the warp, scales one stage ahead (see mxq_grouped.cu) ----------------
        uint32_t count = 0, set = 0;
        bool ok = true, copied = false;
        RingAt<STAGES> at;
        constexpr uint32_t SF_COLS = C::SF_STEPS * 8;
        dependency_wait();                                           // not in a bounded wait while the kernel before this one runs
        const uint32_t idesc = p.idesc | ((uint32_t)(ROWS >> 3) << 17);
        auto copy_scales = [&](int s, uint32_t into) {
            const uint32_t from = ring + s * C::STAGE_BYTES, sfw = tmem + SFW_COL + into, sfx = tmem + SFX_COL + into;
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < C::SF_STEPS; ++c) {
                    tmem_cp_32x128b(sfw + 8 * c, smem_desc(from + C::SFW + c * 512, 0, 128, LAYOUT_NONE));
                    tmem_cp_32x128b(sfx + 8 * c, smem_desc(from + C::SFX + c * 512, 0, 128, LAYOUT_NONE));
                }
            }
            __syncwarp();
        };
        for (int u = u_begin; u < walk.total && ok; u += u_step, ++count) {
            const bool more = u + u_step < walk.total;
            const int a = (int)(count & 1u);
            if (count >= 2) ok = mbar_wait(accum_empty(a), ((count >> 1) - 1) & 1, p.status, ST_MMA_TIMEOUT);
            tc_fence_after();
            const uint32_t d = tmem + a * ACC_STRIDE;
            for (int kt = 0; kt < KT && ok; ++kt, set ^= SF_COLS) {
                const uint32_t st = ring + at.s * C::STAGE_BYTES, empty = empty_bar(at.s);
                if (!copied) {
                    ok = mbar_wait(full_bar(at.s), at.phase, p.status, ST_MMA_TIMEOUT);
                    tc_fence_after();
                    if (!ok) break;
                    copy_scales(at.s, set);
                }
                copied = false;
                at.step();
                if ((kt + 1 < KT || more) && mbar_test_wait(full_bar(at.s), at.phase)) {
                    tc_fence_after();
                    copy_scales(at.s, set ^ SF_COLS);
                    copied = true;
                }
                const uint64_t w_desc = smem_desc(st + C::W, 16, 1024, LAYOUT_SW128), x_desc = smem_desc(st, 16, 1024, LAYOUT_SW128);
                const uint32_t sfw = tmem + SFW_COL + set, sfx = tmem + SFX_COL + set;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t acc = (kt > 0 || k > 0) ? 1u : 0u;
                        if constexpr (MXF4) {
                            const uint32_t id = (k & 1u) * 2u;
                            mma_mxf4(d, w_desc + 2 * k, x_desc + 2 * k, idesc | (id << 29) | (id << 4), sfw + 8 * (k >> 1), sfx + 8 * (k >> 1), acc);
                        } else {
                            mma_mxf8f6f4(d, w_desc + 2 * k, x_desc + 2 * k, idesc | (k << 29) | (k << 4), sfw, sfx, acc);
                        }
                    }
                    mma_commit(empty);
                }
                __syncwarp();
            }
            if (elect_one()) mma_commit(accum_full(a));
            __syncwarp();
        }
        if (!ok) {
            // unwinding after a wait that ran out: the MMAs already issued must finish before tensor memory is freed
            if (elect_one()) mma_commit(drain_bar);
            __syncwarp();
            mbar_wait(drain_bar, 0, nullptr, 0);
        }
    } else if (warp < EPI_WARP || warp >= EPI_WARP + 4) {
        // ---------------- rows: a warp takes every fifth (fourth) stage, 16 lanes a row, two rows at a time ----------------
        constexpr int E = MXF4 ? 16 : 8, WORDS = E * (int)sizeof(T) / 4;                 // elements and words per lane and row
        constexpr int BATCH = 16 / WORDS;                                                // row pairs whose loads are issued together (16 registers)
        constexpr int PAIRS = ROWS / 2;
        using KIn = typename std::conditional<DT == MXQ_F32, KF32, typename std::conditional<DT == MXQ_BF16, KBF16, KF16>::type>::type;
        const int kl = (lane & 15) * E;                                                  // this lane's first element of a step
        const int turn = warp < EPI_WARP ? warp - 2 : warp - EPI_WARP - 2;
        int u = u_begin, kt = turn;
        RingAt<STAGES> at;
        at.step(turn);
        bool ok = true, live = turn < C::QUANT_WARPS, fresh = live;
        Unit t{};
        int from[PAIRS];                                                                 // rows of x; -1: a row of zeros, -2: none
        // the unit of this warp's next stage, and where its rows lie
        auto open = [&]() {
            while (live && kt >= KT) { kt -= KT; u += u_step; fresh = true; live = u < walk.total; }
            live = live && u < walk.total;
            if (!live || !fresh) return;
            fresh = false;
            t = walk.at(u, FEATURES);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int r = 2 * i + (lane >> 4);
                from[i] = r < t.rows ? -1 : -2;
                if (r < t.rows) {
                    int64_t row = t.row + r;
                    if (src.row_index != nullptr)
                        row = src.index64 ? reinterpret_cast<const long long*>(src.row_index)[row] : (int64_t)reinterpret_cast<const int*>(src.row_index)[row];
                    if (row >= 0 && row < src.rows_in) from[i] = (int)row;
                }
            }
        };
        uint32_t w[BATCH][WORDS];
        auto request = [&](int i0) {                                                     // row pairs i0 .. i0 + BATCH - 1 of the stage
            const int k = (k_begin + kt) * C::K_STEP + kl;
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
#pragma unroll
                for (int j = 0; j < WORDS; j += 4) {
                    // a row that does not exist reads as ones (it does not hold up the short form), one outside x as zeros
                    const uint32_t fill = from[i0 + i] == -2 ? one_bits<KIn>() : 0u;
                    uint4 q = make_uint4(fill, fill, fill, fill);
                    if (from[i0 + i] >= 0 && k < p.K)
                        q = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(src.x) + (int64_t)from[i0 + i] * p.K + k) + j / 4);
                    w[i][j] = q.x; w[i][j + 1] = q.y; w[i][j + 2] = q.z; w[i][j + 3] = q.w;
                }
        };
        if (src.row_index != nullptr) dependency_wait();
        open();
        dependency_wait();
        if (live) request(0);
        if (turn < C::QUANT_WARPS && lane == 0) mbar_arrive(rows_bar);
        while (ok && live) {
            const int k = (k_begin + kt) * C::K_STEP + kl, rows = t.rows;
            uint8_t* st = ring_ptr + at.s * C::STAGE_BYTES;
            ok = mbar_wait(empty_bar(at.s), at.phase ^ 1u, p.status, ST_PRODUCER_TIMEOUT);
            if (!ok) break;
            auto quantise = [&](int i0) {
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    if (2 * (i0 + i) >= rows) break;                                     // uniform: neither row of the pair exists
                    uint32_t codes[2];
                    const uint32_t sbyte = quantise_part<KIn, F, OUT, E>(w[i], codes);
                    const int r = 2 * (i0 + i) + (lane >> 4);
                    if (r < rows) {
                        // 8 of the row's 128 bytes: 16-byte unit j lies at j ^ (r % 8)
                        const uint32_t j = (lane & 15) >> 1;
                        *reinterpret_cast<uint2*>(st + r * 128 + ((j ^ (r & 7)) << 4) + (lane & 1) * 8) = make_uint2(codes[0], codes[1]);
                        if (lane % (32 / E) == 0) {
                            // scale of row r and block b at r * 16 + b; blocks behind K are 2^0 (their codes are zero)
                            const int blk = kl / 32;
                            st[C::SFX + (blk >> 2) * 512 + r * 16 + (blk & 3)] = (uint8_t)(k < p.K ? sbyte : 127u);
                        }
                    }
                }
            };
            quantise(0);
#pragma unroll
            for (int i0 = BATCH; i0 < PAIRS; i0 += BATCH) {
                if (2 * i0 >= rows) break;
                request(i0);
                quantise(i0);
            }
            // the next stage's first rows are on their way while this one is handed over and the ring has no room
            kt += C::QUANT_WARPS;
            open();
            if (live) request(0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full_bar(at.s));
            at.step(C::QUANT_WARPS);
        }
    } else if (warp >= EPI_WARP) {
        // ---------------- epilogue: 32 features of 16 rows per warp ----------------
        const int q = warp - EPI_WARP;
        const int er = lane >> 3, ef = q * 32 + (lane & 7) * 4;
        float* slot = slots + q * 512;
        T* out = reinterpret_cast<T*>(p.out);
        const T* extra = reinterpret_cast<const T*>(p.extra);
        const int owner = q / quads;                                                     // the CTA of the cluster that finishes these features
        bool ok = true;
        uint32_t count = 0;
        dependency_wait();
        for (int u = u_begin; u < walk.total && ok; u += u_step, ++count) {
            const Unit t = walk.at(u, FEATURES);
            const int a = (int)(count & 1u), f = t.f0 + ef;
            Four<T> e[4];
            float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (owner == rank) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 4 + er;
                    if (p.extra_mode != X_NONE && r < t.rows) load_four(extra + (size_t)(t.row + r) * p.N + f, p.N - f, p.vector, e[i]);
                }
                if (p.bias != nullptr) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (f + i < p.N) bias[i] = widen(reinterpret_cast<const T*>(p.bias)[(size_t)t.g * p.N + f + i]);
                }
            }
            ok = mbar_wait(accum_full(a), (count >> 1) & 1, p.status, ST_EPILOGUE_TIMEOUT);
            tc_fence_after();
            if (!ok) break;
            uint32_t v[32];
            tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + a * ACC_STRIDE, v);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(accum_empty(a));
            if (split > 1) {
                // a cluster works on one unit: parts are received once.  Part of CTA c for this quadrant: slot c, own one left out
                float* mine = reinterpret_cast<float*>(first + p.rows.groups + 1) + (q % quads) * 512;
                if (owner != rank) {
                    const int place = rank < owner ? rank : rank - 1;
                    const uint32_t to = map_to_rank(smem_u32(mine + place * quads * 512 + lane), (uint32_t)owner);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + j * 128), "r"(v[j]) : "memory");
                    __syncwarp();                                                        // the warp's stores, then their release by one lane
                    if (lane == 0) arrive_at(parts_bar, owner);
                    continue;
                }
                ok = mbar_wait_cluster(parts_bar, 0, p.status, ST_EPILOGUE_TIMEOUT);
                if (!ok) break;
                float sum[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[j] = 0.0f;
                for (int c = 0; c < split; ++c) {                                        // in the order of the CTAs
                    const float* part = mine + (c < rank ? c : c - 1) * quads * 512;
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[j] += c == rank ? __uint_as_float(v[j]) : part[j * 32 + lane];
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(sum[j]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) slot[j * 32 + lane] = __uint_as_float(v[j]);
            __syncwarp();
            T* at = out + (size_t)(t.row + er) * p.N + f;
            const int rows = (t.rows - er + 3) >> 2, left = p.N - f;
            finish_any(p.act, slot, lane, bias, e, p.extra_mode, at, p.N, rows, left, p.vector);
            __syncwarp();
        }
        if (p.zero_rest) zero_rows_outside(out, first[0], first[p.rows.groups], p.rows.rows, p.N, threadIdx.x - EPI_WARP * 32, 128);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
    if (split > 1) cluster_barrier();                                // no CTA leaves while another may still write to it
}

template <int DT, class F, int OUT>
static int launch(const Params& p, const Source& src, int split, cudaStream_t st) {
    using C = Cfg<OUT == 5>;
    static bool attr_done[MAX_DEVICES] = {false};
    const cudaError_t e = raise_smem_limit(decode_kernel<DT, F, OUT>, C::smem_bytes(MAX_GROUPS, 2), attr_done);
    if (e != cudaSuccess) { set_last_cuda_error(e); return MXQ_ELAUNCH; }
    const int64_t units = most_units(p.rows, p.N, FEATURES), room = 2 * sm_count();
    // a cluster works on one unit; without clusters the CTAs stay and walk over theirs
    return launch_after(decode_kernel<DT, F, OUT>, (unsigned)(split > 1 ? units * split : units < room ? units : room), THREADS, C::smem_bytes(p.rows.groups, split),
                        (unsigned)split, st, p, src, split);
}

}  // namespace decode

int decode_rows() { return decode::ROWS; }

int launch_decode(const Params& p, int dt, const void* x, const void* row_index, int index64, int64_t rows_in, int eb, int fb, bool nibbles,
                  cudaStream_t st) {
    // CTAs that share a unit: as many as the SMs hold (two each, beside a large table one), the steps of K allow, and 4 at most (a lane quadrant each)
    const int64_t units = most_units(p.rows, p.N, decode::FEATURES);
    const int steps = (p.K + (nibbles ? 255 : 127)) / (nibbles ? 256 : 128);
    int split = 1;
    const int64_t room = (int64_t)sm_count() * (nibbles ? decode::Cfg<true>::per_sm(p.rows.groups, 2) : decode::Cfg<false>::per_sm(p.rows.groups, 2));
    while (split < 4 && units * split * 2 <= room && steps >= split * 2 * 4) split *= 2;
    const decode::Source src{x, row_index, index64, rows_in};
    int rc = MXQ_ESIZE;
    with_row_format(eb, fb, nibbles, [&](auto fmt, auto out) {
        using F = decltype(fmt);
        constexpr int OUT = decltype(out)::value;
        if (dt == MXQ_F32) rc = decode::launch<MXQ_F32, F, OUT>(p, src, split, st);
        else if (dt == MXQ_BF16) rc = decode::launch<MXQ_BF16, F, OUT>(p, src, split, st);
        else rc = decode::launch<MXQ_F16, F, OUT>(p, src, split, st);
    });
    return rc;
}

}  // namespace grouped
}  // namespace mxq
