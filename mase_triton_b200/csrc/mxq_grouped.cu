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
//   * the rows' scales lie in memory as one 32-bit word (four blocks) per row and 128 elements of K, the words of
//     consecutive rows side by side; a warp gathers those of a tile into the 512-byte chunks that tcgen05.cp expects,
//     so that no layout depends on where the groups begin;
//   * an accumulator holds a feature per lane and a row per column: bias is one value per lane, and the 32 lanes of a
//     warp read the second operand and write the result 32 consecutive features at a time.
// Which rows belong to which group is read on the device: no size but the upper bounds is known to the host.
//
// Operand layout in HBM:
//   weights: codes [groups * N, K] (bytes, or nibbles for E2M1 x E2M1), scales per group as for a left operand of mxq_gemm.cu
//            ([ceil(N / 256)][ceil(K / 128)][2][512] bytes);
//   rows:    codes [rows, K], scales [ceil(K / 128)][pitch] words, pitch = rows rounded up to 4.
#include <cmath>

#include "mxq_codec.h"
#include "mxq_tc.cuh"

namespace mxq {
namespace grouped {

using namespace tc;

constexpr int MAX_GROUPS = MX_MAX_GROUPS;
constexpr int EPI_WARPS = 8;                     // two per TMEM lane quadrant
constexpr int FIRST_EPI_WARP = 4;                // warps 0..2: TMA producer, MMA issuer, scale gatherer
constexpr int THREADS = (FIRST_EPI_WARP + EPI_WARPS) * 32;

enum : int { X_NONE = MXQ_EXTRA_NONE, X_MUL = MXQ_EXTRA_MULTIPLY, X_ADD = MXQ_EXTRA_ADD };

// MH: 128-feature halves of a tile; BT: widest row tile; MXF4: both operands packed E2M1 nibbles (256 elements of K per 128 bytes)
template <int MH_, int BT_, int STAGES_, bool MXF4_> struct Cfg {
    static constexpr int MH = MH_, BT = BT_, STAGES = STAGES_;
    static constexpr bool MXF4 = MXF4_;
    static constexpr int FEATURES = 128 * MH;
    static constexpr int K_STEP = MXF4 ? 256 : 128;                 // elements of K per stage
    static constexpr int SF_STEPS = MXF4 ? 2 : 1;                   // 128-element steps of scales per stage
    static constexpr int W_BYTES = FEATURES * 128, X_BYTES = BT * 128;
    static constexpr int X_CHUNKS = BT > 128 ? 2 : 1;
    static constexpr int SF_STEP_BYTES = (MH + X_CHUNKS) * 512;
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + SF_STEPS * SF_STEP_BYTES;
    // Two accumulators of BT columns.  MH = 2: the two halves of one tile.  MH = 1: two tiles in turn, so that one is read
    // while the next is computed.  They begin at multiples of 32 columns; the scales take the columns behind them.
    static constexpr int ACC_STRIDE = (BT + 31) / 32 * 32;
    static constexpr int SFW_COL = ACC_STRIDE > BT ? BT : 2 * ACC_STRIDE;
    static constexpr int SFX_COL = ACC_STRIDE > BT ? ACC_STRIDE + BT : SFW_COL + SF_STEPS * 8;
    static_assert(ACC_STRIDE == BT || SFW_COL + SF_STEPS * 8 <= ACC_STRIDE, "tensor memory");
    static_assert(SFX_COL + SF_STEPS * 8 <= 512, "tensor memory");
    static_assert(STAGE_BYTES % 1024 == 0, "the 128-byte swizzle repeats every 1024 bytes");
    static constexpr int TABLE_BYTES = 2 * (MAX_GROUPS + 1) * 4;
    static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 256 + TABLE_BYTES;
    static_assert(SMEM_BYTES <= 232448, "more shared memory than a CTA can have");
};
using Wide = Cfg<2, 240, 3, false>;
using WideFp4 = Cfg<2, 240, 3, true>;
using Narrow = Cfg<1, 128, 6, false>;
using NarrowFp4 = Cfg<1, 128, 6, true>;

struct Params {
    const uint8_t* w_sf;         // weight scales, w_sf_group bytes per group
    int64_t w_sf_group;
    const uint32_t* x_sf;        // row scales
    int64_t x_sf_pitch;          // words per 128-element step of K
    void* out;
    const void* bias;            // [groups, N] or null
    const void* extra;           // [rows, N] or null
    const void* offsets;         // [groups + 1], or null: one group of all rows
    int offsets64;
    int rows, groups, N, K;
    int width;                   // rows per tile at most (a multiple of 16, <= BT)
    int act, extra_mode;
    int zero_rest;               // write zeros into the rows that belong to no group
    uint32_t idesc;              // instruction descriptor without the width
    int* status;
};

template <int DT> struct Elem;
template <> struct Elem<MXQ_F32> { typedef float T; };
template <> struct Elem<MXQ_BF16> { typedef __nv_bfloat16 T; };
template <> struct Elem<MXQ_F16> { typedef __half T; };
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(float v, __half& o) { o = __float2half_rn(v); }

// z * sigmoid(2u) is 0.5 z (1 + tanh u); exp overflows to Inf for very negative arguments and the quotient is then 0
__device__ __forceinline__ float sigmoid_times(float z, float a) { return __fdividef(z, 1.0f + __expf(-a)); }
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case MXQ_ACT_RELU: return z < 0.0f ? 0.0f : z;                       // NaN stays NaN
        case MXQ_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case MXQ_ACT_GELU_TANH: return sigmoid_times(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
        case MXQ_ACT_SILU: return sigmoid_times(z, z);
        default: return z;
    }
}

// where a unit of work lies: features [f0, f0 + FEATURES) of group g for rows [row, row + rows)
struct Unit {
    int g, f0, ftile, row, rows;
    __device__ __forceinline__ uint32_t padded() const { return (uint32_t)(rows + 15) & ~15u; }
};

// The group table (tile counts summed over the groups, first rows) and the walk over the units of one CTA.
struct Walk {
    const int *tiles, *first;
    int g, ftiles, width, total;
    __device__ __forceinline__ Walk(const int* t, const int* f, int groups, int ftiles_, int width_)
        : tiles(t), first(f), g(0), ftiles(ftiles_), width(width_), total(t[groups] * ftiles_) {}
    __device__ __forceinline__ Unit at(int u, int features) {
        while (u >= tiles[g + 1] * ftiles) ++g;                              // units are visited in rising order
        const int tt = tiles[g + 1] - tiles[g], begin = first[g], n = first[g + 1] - begin;
        int ti, fi;
        tile_coords(u - tiles[g] * ftiles, tt, ftiles, ti, fi);
        // tiles of equal width: ceil(n / tt) rounded up to 16 is at most `width`, and the last tile is never empty
        const int w = ((n + tt - 1) / tt + 15) & ~15;
        return Unit{g, fi * features, fi, begin + ti * w, min(w, n - ti * w)};
    }
};

__device__ __forceinline__ int offset_at(const Params& p, int i) {
    if (p.offsets == nullptr) return i == 0 ? 0 : p.rows;
    const int64_t v = p.offsets64 ? reinterpret_cast<const long long*>(p.offsets)[i] : (int64_t)reinterpret_cast<const int*>(p.offsets)[i];
    return (int)min(max(v, (int64_t)0), (int64_t)p.rows);
}

// One warp: first[i] = the largest of offsets[0 .. i] (offsets that fall back leave an empty group and never an overlap),
// tiles[i] = row tiles of the groups before i.
__device__ __forceinline__ void build_table(const Params& p, int* tiles, int* first, int lane) {
    int high = 0, sum = 0;
    for (int base = 0; base <= p.groups; base += 32) {
        const int i = base + lane;
        int v = i <= p.groups ? offset_at(p, i) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(~0u, v, o); if (lane >= o) v = max(v, up); }
        v = max(v, high);
        const int before = __shfl_up_sync(~0u, v, 1);
        // rows of group i - 1, which the running sum at i counts
        int t = (i == 0 || i > p.groups) ? 0 : ((v - (lane == 0 ? high : before)) + p.width - 1) / p.width;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(~0u, t, o); if (lane >= o) t += up; }
        t += sum;
        if (i <= p.groups) { first[i] = v; tiles[i] = t; }
        high = __shfl_sync(~0u, v, 31);
        sum = __shfl_sync(~0u, t, 31);
    }
}

template <class C, int DT>
__global__ void __launch_bounds__(THREADS, 1)
grouped_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x64, const __grid_constant__ CUtensorMap map_x16,
               const __grid_constant__ Params p) {
    constexpr int MH = C::MH, STAGES = C::STAGES;
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

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }      // full: the copies and the gathered scales
        for (int a = 0; a < 2; ++a) { mbar_init(accum_full(a), 1); mbar_init(accum_empty(a), EPI_WARPS); }
        mbar_init(drain_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 3) build_table(p, tiles, first, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int KT = (p.K + C::K_STEP - 1) / C::K_STEP, KT128 = (p.K + 127) / 128;
    const int ftiles = (p.N + C::FEATURES - 1) / C::FEATURES;
    Walk walk(tiles, first, p.groups, ftiles, p.width);
    auto halves_of = [&](const Unit& t) { return MH == 2 && p.N - t.f0 > 128 ? 2 : 1; };

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        bool ok = true;
        uint32_t it = 0;
        for (int u = blockIdx.x; u < walk.total && ok; u += gridDim.x) {
            const Unit t = walk.at(u, C::FEATURES);
            const int halves = halves_of(t);
            const uint32_t n = t.padded();
            const uint8_t* sf = p.w_sf + (size_t)t.g * p.w_sf_group +
                                (MH == 2 ? (size_t)t.ftile * KT128 * 1024 : (size_t)(t.ftile >> 1) * KT128 * 1024 + (t.ftile & 1) * 512);
            const int w_row = t.g * p.N + t.f0;
            const uint32_t tx = (uint32_t)halves * (16384u + C::SF_STEPS * 512u) + n * 128u;
            for (int kt = 0; kt < KT && ok; ++kt, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES) ok = mbar_wait(empty_bar(s), ((it / STAGES) & 1) ^ 1, p.status, ST_PRODUCER_TIMEOUT);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t st = ring + s * C::STAGE_BYTES;
                    mbar_expect_tx(full_bar(s), tx);
                    for (int h = 0; h < halves; ++h) tma_load_2d(st + h * 16384, &map_w, kt * C::K_STEP, w_row + h * 128, full_bar(s));
                    uint32_t r = 0;
                    for (; r + 64 <= n; r += 64) tma_load_2d(st + C::W_BYTES + r * 128, &map_x64, kt * C::K_STEP, t.row + r, full_bar(s));
                    for (; r < n; r += 16) tma_load_2d(st + C::W_BYTES + r * 128, &map_x16, kt * C::K_STEP, t.row + r, full_bar(s));
#pragma unroll
                    for (int c = 0; c < C::SF_STEPS; ++c)
                        bulk_load(st + C::W_BYTES + C::X_BYTES + c * C::SF_STEP_BYTES, sf + (size_t)(kt * C::SF_STEPS + c) * 1024, halves * 512, full_bar(s));
                }
                __syncwarp();
            }
        }
        // every copy this warp started must have landed before the CTA gives its shared memory back (returns at once in a run that went well)
        for (uint32_t j = it > (uint32_t)STAGES ? it - STAGES : 0u; j < it; ++j)
            mbar_wait(full_bar(j % STAGES), (j / STAGES) & 1, p.status, ST_PRODUCER_TIMEOUT);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        bool ok = true;
        uint32_t it = 0, count = 0;
        for (int u = blockIdx.x; u < walk.total && ok; u += gridDim.x, ++count) {
            const Unit t = walk.at(u, C::FEATURES);
            const int halves = halves_of(t);
            const uint32_t n = t.padded();
            const uint32_t idesc_n = p.idesc | ((n >> 3) << 17);
            const int buf = MH == 1 ? (int)(count & 1u) : 0;
            for (int kt = 0; kt < KT && ok; ++kt, ++it) {
                const int s = it % STAGES;
                ok = mbar_wait(full_bar(s), (it / STAGES) & 1, p.status, ST_MMA_TIMEOUT);
                const uint32_t st = ring + s * C::STAGE_BYTES, sf = st + C::W_BYTES + C::X_BYTES;
                const uint64_t x_desc = smem_desc(st + C::W_BYTES, 16, 1024, LAYOUT_SW128);
                for (int h = 0; h < halves; ++h) {
                    const int a = MH == 1 ? buf : h;
                    // the first product into an accumulator overwrites it: the epilogue must have read what it held
                    if (kt == 0 && ok) {
                        if constexpr (MH == 1) { if (count >= 2) ok = mbar_wait(accum_empty(a), ((count >> 1) - 1) & 1, p.status, ST_MMA_TIMEOUT); }
                        else { if (count >= 1) ok = mbar_wait(accum_empty(a), (count - 1) & 1, p.status, ST_MMA_TIMEOUT); }
                    }
                    tc_fence_after();
                    if (ok && lane == 0) {
                        if (h == 0) {
#pragma unroll
                            for (int c = 0; c < C::SF_STEPS; ++c) {
                                const uint32_t src = sf + c * C::SF_STEP_BYTES;
                                for (int hh = 0; hh < halves; ++hh)
                                    tmem_cp_32x128b(tmem + C::SFW_COL + 8 * c + 4 * hh, smem_desc(src + 512 * hh, 0, 128, LAYOUT_NONE));
                                tmem_cp_32x128b(tmem + C::SFX_COL + 8 * c, smem_desc(src + MH * 512, 0, 128, LAYOUT_NONE));
                                if (C::X_CHUNKS == 2 && n > 128)
                                    tmem_cp_32x128b(tmem + C::SFX_COL + 8 * c + 4, smem_desc(src + MH * 512 + 512, 0, 128, LAYOUT_NONE));
                            }
                        }
                        const uint64_t w_desc = smem_desc(st + h * 16384, 16, 1024, LAYOUT_SW128);
                        const uint32_t d = tmem + a * C::ACC_STRIDE;
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) {
                            const uint32_t acc = (kt > 0 || k > 0) ? 1u : 0u;
                            if constexpr (C::MXF4) {
                                const uint32_t id = (k & 1u) * 2u;                 // 64 elements: scale bytes (0, 1) or (2, 3) of step k / 2
                                mma_mxf4(d, w_desc + 2 * k, x_desc + 2 * k, idesc_n | (id << 29) | (id << 4),
                                         tmem + C::SFW_COL + 8 * (k >> 1) + 4 * h, tmem + C::SFX_COL + 8 * (k >> 1), acc);
                            } else {
                                mma_mxf8f6f4(d, w_desc + 2 * k, x_desc + 2 * k, idesc_n | (k << 29) | (k << 4),
                                             tmem + C::SFW_COL + 4 * h, tmem + C::SFX_COL, acc);
                            }
                        }
                        if (h == halves - 1) mma_commit(empty_bar(s));
                    }
                    __syncwarp();
                }
            }
            if (lane == 0) mma_commit(accum_full(buf));
            __syncwarp();
        }
        if (!ok) {
            // unwinding after a wait that ran out: the MMAs already issued must finish before tensor memory is freed
            if (lane == 0) mma_commit(drain_bar);
            __syncwarp();
            mbar_wait(drain_bar, 0, nullptr, 0);
        }
    } else if (warp == 2) {
        // ---------------- scales of the rows: words of consecutive rows -> chunks ----------------
        // chunk c of a tile: rows 128c .. 128c + 127, the word of row r at (r % 32) * 16 + (r / 32) * 4: lane l owns rows l, l + 32, ...
        bool ok = true;
        uint32_t it = 0;
        for (int u = blockIdx.x; u < walk.total && ok; u += gridDim.x) {
            const Unit t = walk.at(u, C::FEATURES);
            const int chunks = C::X_CHUNKS == 2 && t.rows > 128 ? 2 : 1;
            for (int kt = 0; kt < KT && ok; ++kt, ++it) {
                const int s = it % STAGES;
                uint32_t w[C::SF_STEPS * C::X_CHUNKS][4];
#pragma unroll
                for (int c = 0; c < C::SF_STEPS; ++c) {
                    const uint32_t* src = p.x_sf + (size_t)(kt * C::SF_STEPS + c) * p.x_sf_pitch;
#pragma unroll
                    for (int ch = 0; ch < C::X_CHUNKS; ++ch)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = ch * 128 + j * 32 + lane;
                            w[c * C::X_CHUNKS + ch][j] = r < t.rows ? __ldcg(src + t.row + r) : 0x7F7F7F7Fu;
                        }
                }
                if (it >= STAGES) ok = mbar_wait(empty_bar(s), ((it / STAGES) & 1) ^ 1, p.status, ST_PRODUCER_TIMEOUT);
                if (!ok) break;
                uint8_t* dst = ring_ptr + s * C::STAGE_BYTES + C::W_BYTES + C::X_BYTES + MH * 512;
#pragma unroll
                for (int c = 0; c < C::SF_STEPS; ++c)
                    for (int ch = 0; ch < chunks; ++ch) {
                        const uint32_t* v = w[c * C::X_CHUNKS + ch];
                        *reinterpret_cast<uint4*>(dst + c * C::SF_STEP_BYTES + ch * 512 + lane * 16) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(s));
            }
        }
    } else if (warp >= FIRST_EPI_WARP) {
        // ---------------- epilogue ----------------
        typedef typename Elem<DT>::T T;
        const int q = warp & 3, side = (warp - FIRST_EPI_WARP) >> 2;      // lane quadrant; the two warps of one take 16-row chunks in turn
        T* out = reinterpret_cast<T*>(p.out);
        const T* extra = reinterpret_cast<const T*>(p.extra);
        bool ok = true;
        uint32_t count = 0;
        for (int u = blockIdx.x; u < walk.total && ok; u += gridDim.x, ++count) {
            const Unit t = walk.at(u, C::FEATURES);
            const int halves = halves_of(t);
            const int buf = MH == 1 ? (int)(count & 1u) : 0;
            ok = mbar_wait(accum_full(buf), MH == 1 ? (count >> 1) & 1 : count & 1, p.status, ST_EPILOGUE_TIMEOUT);
            tc_fence_after();
            if (!ok) break;
            const int chunks = (t.rows + 15) >> 4;
            for (int h = 0; h < MH; ++h) {
                const int a = MH == 1 ? buf : h;
                const int f = t.f0 + h * 128 + q * 32 + lane;
                const bool live = h < halves && f < p.N;
                const float b = (p.bias != nullptr && live) ? widen(reinterpret_cast<const T*>(p.bias)[(size_t)t.g * p.N + f]) : 0.0f;
                if (h < halves) {
                    for (int c = side; c < chunks; c += 2) {
                        uint32_t r[32];
                        tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + a * C::ACC_STRIDE + c * 16, r);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        const int n = min(16, t.rows - c * 16);
                        const size_t at = (size_t)(t.row + c * 16) * p.N + f;
                        T e[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (p.extra_mode != X_NONE && live && j < n) e[j] = extra[at + (size_t)j * p.N];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if (!live || j >= n) continue;
                            float y = activate(__uint_as_float(r[j]) + b, p.act);
                            if (p.extra_mode == X_MUL) y *= widen(e[j]);
                            else if (p.extra_mode == X_ADD) y += widen(e[j]);
                            T o;
                            narrow(y, o);
                            out[at + (size_t)j * p.N] = o;
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(accum_empty(a));
            }
        }
        if (p.zero_rest) {
            // rows before the first group and behind the last one
            const int lo = first[0], hi = first[p.groups];
            const int64_t rest = (int64_t)(lo + p.rows - hi) * p.N;
            for (int64_t i = (int64_t)blockIdx.x * (EPI_WARPS * 32) + (threadIdx.x - FIRST_EPI_WARP * 32); i < rest; i += (int64_t)gridDim.x * (EPI_WARPS * 32)) {
                const int64_t before = (int64_t)lo * p.N;
                narrow(0.0f, out[i < before ? i : i - before + (int64_t)hi * p.N]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
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

// One thread per row and 32-element block, padding blocks of the last 128 elements included (scale 2^0; the copies fill their
// codes with zeros).  A row index outside x gives a row of zeros.
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint8_t* __restrict__ scales, const uint8_t* __restrict__ elements,
                                                        const void* __restrict__ row_index, int index64, int64_t rows_in, int64_t rows,
                                                        int K, int nibbles, uint8_t* __restrict__ codes, uint8_t* __restrict__ sf, int64_t sf_pitch,
                                                        const __grid_constant__ CodeTables t) {
    __shared__ uint8_t s_plain[256], s_halved[256];
    s_plain[threadIdx.x] = t.plain[threadIdx.x];
    s_halved[threadIdx.x] = t.halved[threadIdx.x];
    __syncthreads();
    const int blocks = (K + 127) / 128 * 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * blocks) return;
    const int64_t row = i / blocks;
    const int kb = (int)(i - row * blocks);
    uint8_t* sf_at = sf + ((int64_t)(kb >> 2) * sf_pitch + row) * 4 + (kb & 3);
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
    if (nibbles) {
        uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j >> 3] |= (uint32_t)(cb[j] & 0xFu) << (4 * (j & 7));
        *reinterpret_cast<uint4*>(codes + row * (K / 2) + kb * 16) = make_uint4(o[0], o[1], o[2], o[3]);
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
    uint4* to = reinterpret_cast<uint4*>(codes + row * K + kb * 32);
    to[0] = o[0];
    to[1] = o[1];
    *sf_at = (uint8_t)((any_bad && scale < 255u) ? scale + 1u : scale);
}

// box of `box_rows` rows x 128 bytes of a [rows, K] operand
static bool make_map(CUtensorMap* map, const void* codes, int64_t rows, int64_t K, int box_rows, bool nibbles) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(nibbles ? K / 2 : K)};
    const cuuint32_t box[2] = {(cuuint32_t)(nibbles ? 256 : 128), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, nibbles ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN8B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class C, int DT>
static int launch(const Params& p, const uint8_t* w_codes, const uint8_t* x_codes, cudaStream_t st) {
    static bool attr_done[MAX_DEVICES] = {false};
    const cudaError_t e = raise_smem_limit(grouped_kernel<C, DT>, C::SMEM_BYTES, attr_done);
    if (e != cudaSuccess) { set_last_cuda_error(e); return MXQ_ELAUNCH; }
    CUtensorMap mw, mx64, mx16;
    if (!make_map(&mw, w_codes, (int64_t)p.groups * p.N, p.K, 128, C::MXF4) || !make_map(&mx64, x_codes, p.rows, p.K, 64, C::MXF4) ||
        !make_map(&mx16, x_codes, p.rows, p.K, 16, C::MXF4)) return MXQ_ELAUNCH;
    // units at most: every group may end in a partial tile; what the groups leave is known on the device only
    const int64_t ftiles = (p.N + C::FEATURES - 1) / C::FEATURES;
    const int64_t most = (int64_t)(p.rows / p.width + (p.groups < p.rows ? p.groups : p.rows)) * ftiles;
    const int grid = (int)(most < sm_count() ? most : sm_count());
    grouped_kernel<C, DT><<<grid, THREADS, C::SMEM_BYTES, st>>>(mw, mx64, mx16, p);
    return check_launch();
}

template <class C>
static int launch_dt(Params& p, int dt, const uint8_t* w_codes, const uint8_t* x_codes, cudaStream_t st) {
    if (p.width == 0 || p.width > C::BT) p.width = C::BT;
    if (dt == MXQ_F32) return launch<C, MXQ_F32>(p, w_codes, x_codes, st);
    if (dt == MXQ_BF16) return launch<C, MXQ_BF16>(p, w_codes, x_codes, st);
    return launch<C, MXQ_F16>(p, w_codes, x_codes, st);
}

static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
static int64_t sf_pitch(int64_t rows) { return (rows + 3) / 4 * 4; }

}  // namespace grouped
}  // namespace mxq

using namespace mxq;

extern "C" int mxq_mx_max_groups(void) { return grouped::MAX_GROUPS; }

extern "C" int64_t mxq_mx_grouped_scratch_bytes(int64_t rows_in, int64_t rows, int64_t K) {
    if (rows_in < 0 || rows < 0 || K <= 0 || K % 32 != 0) return MXQ_EINVAL;
    return grouped::align256(rows * K) + grouped::align256((K + 127) / 128 * grouped::sf_pitch(rows) * 4) + grouped::align256(rows_in * K) +
           grouped::align256(rows_in * K / 32);
}

extern "C" int mxq_mx_grouped_linear(const void* x, int x_dtype, int64_t rows_in, int64_t rows, int64_t K, int x_exp_bits, int x_frac_bits,
                                     int x_round_mode, const void* row_index, int index64, const uint8_t* w_codes, const uint8_t* w_sf,
                                     int w_hw_format, int64_t groups, int64_t N, const void* offsets, int offsets64, void* out, const void* bias,
                                     int activation, const void* extra, int extra_mode, int zero_rest, void* scratch, int64_t scratch_bytes,
                                     int* status, void* stream) {
    if (rows < 0 || rows_in < 0 || groups <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return MXQ_EINVAL;
    if (x_dtype != MXQ_F32 && x_dtype != MXQ_BF16 && x_dtype != MXQ_F16) return MXQ_EINVAL;
    if (activation < MXQ_ACT_NONE || activation > MXQ_ACT_SILU || extra_mode < MXQ_EXTRA_NONE || extra_mode > MXQ_EXTRA_ADD) return MXQ_EINVAL;
    if (row_index == nullptr && rows != rows_in) return MXQ_EINVAL;
    if (offsets == nullptr && groups != 1) return MXQ_EINVAL;
    if (groups > grouped::MAX_GROUPS || rows > (1 << 30) || N > (1 << 30) || K > (1 << 30) || groups * N > (1ll << 31) - 1) return MXQ_ESIZE;
    if (rows * ((K + 127) / 128 * 4) > (1ll << 31) * 255 || rows_in > (1 << 30)) return MXQ_ESIZE;
    if (rows == 0) return MXQ_OK;
    if ((!x && rows_in > 0) || !w_codes || !w_sf || !out || !scratch || (extra_mode != MXQ_EXTRA_NONE && !extra)) return MXQ_EINVAL;
    if ((reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(w_sf)) % 16 != 0 || reinterpret_cast<uintptr_t>(scratch) % 256 != 0) return MXQ_EINVAL;
    if (scratch_bytes < mxq_mx_grouped_scratch_bytes(rows_in, rows, K)) return MXQ_ESIZE;
    // both operands E2M1 and the weight kept as nibbles: the 4-bit kind
    const bool x_e2m1 = x_exp_bits == 2 && x_frac_bits == 1;
    const bool fp4 = w_hw_format == 5;
    if (fp4 && (!x_e2m1 || K % 256 != 0 || reinterpret_cast<uintptr_t>(w_codes) % 32 != 0)) return MXQ_EINVAL;
    if (!fp4 && w_hw_format != 0 && w_hw_format != 1) return MXQ_EINVAL;
    grouped::CodeTables tables;
    int x_fmt = 0;
    if (!hw_code_tables(x_exp_bits, x_frac_bits, tables.plain, tables.halved, tables.bad, &x_fmt)) return MXQ_EINVAL;

    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* sf = codes + grouped::align256(rows * K);
    uint8_t* ref_codes = sf + grouped::align256((K + 127) / 128 * grouped::sf_pitch(rows) * 4);
    uint8_t* ref_scales = ref_codes + grouped::align256(rows_in * K);
    cudaStream_t st = (cudaStream_t)stream;
    if (rows_in > 0) {
        const int rc = mxq_mxfp_extract(x, x_dtype, ref_scales, ref_codes, rows_in * K, 32, x_exp_bits, x_frac_bits, 1, x_round_mode, stream);
        if (rc != MXQ_OK) return rc;
    }
    const int64_t threads = rows * ((K + 127) / 128 * 4);
    grouped::pack_rows_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(ref_scales, ref_codes, row_index, index64, rows_in, rows, (int)K, fp4, codes, sf,
                                                                                grouped::sf_pitch(rows), tables);
    const int rc = check_launch();
    if (rc != MXQ_OK) return rc;

    grouped::Params p{};
    p.w_sf = w_sf;
    p.w_sf_group = mxq_mx_sf_bytes(N, K, MXQ_OPERAND_A, 0);
    p.x_sf = reinterpret_cast<const uint32_t*>(sf);
    p.x_sf_pitch = grouped::sf_pitch(rows);
    p.out = out; p.bias = bias; p.extra = extra; p.offsets = offsets; p.offsets64 = offsets64;
    p.rows = (int)rows; p.groups = (int)groups; p.N = (int)N; p.K = (int)K;
    p.act = activation; p.extra_mode = extra_mode; p.zero_rest = zero_rest; p.status = status;
    // formats of left (weight) and right (rows) operand, K-major both, E8M0 scales, M >> 4; E2M1 is 1 in the 4-bit kind's encoding
    p.idesc = (fp4 ? (1u << 7) | (1u << 10) : ((uint32_t)w_hw_format << 7) | ((uint32_t)x_fmt << 10)) | (1u << 23) | ((uint32_t)(128 >> 4) << 24);
    const bool narrow = rows / groups <= 128;
    if (fp4) return narrow ? grouped::launch_dt<grouped::NarrowFp4>(p, x_dtype, w_codes, codes, st) : grouped::launch_dt<grouped::WideFp4>(p, x_dtype, w_codes, codes, st);
    return narrow ? grouped::launch_dt<grouped::Narrow>(p, x_dtype, w_codes, codes, st) : grouped::launch_dt<grouped::Wide>(p, x_dtype, w_codes, codes, st);
}
