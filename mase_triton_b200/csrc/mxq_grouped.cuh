// Pieces shared by the kernels of the grouped products (mxq_grouped.cu, mxq_grouped_decode.cu): the group table and the walk over
// the units of work, the epilogue's arithmetic, launches that may overlap the kernel before them.
#pragma once
#include "mxq_quant.cuh"
#include "mxq_tc.cuh"

namespace mxq {
namespace grouped {

using namespace tc;

constexpr int MAX_GROUPS = MX_MAX_GROUPS;
enum : int { X_NONE = MXQ_EXTRA_NONE, X_MUL = MXQ_EXTRA_MULTIPLY, X_ADD = MXQ_EXTRA_ADD };

// Packed weights: 128 features x one step of K (128 bytes of codes per feature: 128 elements, 256 of E2M1 pairs) are one contiguous
// block, the codes as the 128-byte-swizzled image that the tensor cores read in shared memory, their scale chunks behind
// them.  [group][ceil(N / 128)][steps of K] blocks: a CTA reads a sequential stream with plain bulk copies.  (Codes in rows, fetched in boxes
// of 128 rows x 128 bytes, cost a DRAM page per line: see the measurements in mxq_grouped_decode.cu.)
template <bool MXF4> struct WeightTile {
    static constexpr int K_STEP = MXF4 ? 256 : 128, SF_STEPS = MXF4 ? 2 : 1;
    static constexpr int CODES = 16384, BYTES = CODES + SF_STEPS * 512;
    static __host__ __device__ int64_t steps(int64_t K) { return (K + K_STEP - 1) / K_STEP; }
    static __host__ __device__ int64_t group_bytes(int64_t N, int64_t K) { return (N + 127) / 128 * steps(K) * BYTES; }
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

// Four consecutive features of a row as one 8-byte (fp32: 16-byte) access; `left` of the row's features begin here, `vector`: rows and
// base are aligned to four.  Held as words: a struct of four 16-bit values is copied member by member, i.e. in 2-byte accesses.
template <class T> struct Words { typedef uint2 V; };
template <> struct Words<float> { typedef uint4 V; };
template <class T> union Four {
    typename Words<T>::V w;
    T v[4];
    __device__ __forceinline__ Four() {}
};
template <class T> __device__ __forceinline__ void load_four(const T* at, int left, int vector, Four<T>& o) {
    if (vector) { if (left > 0) o.w = __ldcg(reinterpret_cast<const typename Words<T>::V*>(at)); return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (k < left) o.v[k] = at[k];
}
template <class T> __device__ __forceinline__ void store_four(T* at, int left, int vector, const Four<T>& o) {
    if (vector) { if (left > 0) *reinterpret_cast<typename Words<T>::V*>(at) = o.w; return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (k < left) at[k] = o.v[k];
}

// z sigmoid(a), the tail included: with t = exp(-|a|) the divisor lies in [1, 2], where the fast division holds (beyond 2^126 it gives 0), and
// nothing overflows.  For fp32 results expf: in __expf the rounding of a log2(e) alone costs |a| half steps of 2^-24.  16-bit results have
// steps of 2^-11 at least, beside at most 104 of those half steps where t is not 0: __expf (expf: 8192 x 4096 x 14336 532 -> 551 us).
// (z sigmoid(2u) is 0.5 z (1 + tanh u).)
template <class T> __device__ __forceinline__ float sigmoid_times(float z, float a) {
    const float t = sizeof(T) == 4 ? expf(-fabsf(a)) : __expf(-fabsf(a));
    return __fdividef(a < 0.0f ? z * t : z, 1.0f + t);
}
template <int ACT, class T> __device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == MXQ_ACT_RELU) return z < 0.0f ? 0.0f : z;                       // NaN stays NaN
    else if constexpr (ACT == MXQ_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    else if constexpr (ACT == MXQ_ACT_GELU_TANH) return sigmoid_times<T>(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
    else if constexpr (ACT == MXQ_ACT_SILU) return sigmoid_times<T>(z, z);
    else return z;
}
// The epilogue of one lane's 4 x 4 values: rows at, at + 4 * pitch, ... (`rows` of them exist, at most four), four features each.
// The choices are made once for all sixteen: a switch per value costs more than the values.
template <int ACT, class T>
__device__ __forceinline__ void finish(const float* slot, int lane, const float (&bias)[4], const Four<T> (&extra)[4], int extra_mode, T* at, int64_t pitch, int rows,
                                       int left, int vector) {
    float y[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 v = reinterpret_cast<const float4*>(slot)[i * 32 + lane];
        y[4 * i] = v.x; y[4 * i + 1] = v.y; y[4 * i + 2] = v.z; y[4 * i + 3] = v.w;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) y[k] = activate<ACT, T>(y[k] + bias[k & 3]);
    if (extra_mode == X_MUL) {
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] *= widen(extra[k >> 2].v[k & 3]);
    } else if (extra_mode == X_ADD) {
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] += widen(extra[k >> 2].v[k & 3]);
    }
    Four<T> o[4];
#pragma unroll
    for (int k = 0; k < 16; ++k) narrow(y[k], o[k >> 2].v[k & 3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < rows) store_four(at + i * 4 * pitch, left, vector, o[i]);
}

// a value that every lane holds, in a uniform register
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(~0u, v, 0); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(~0u, v, 0); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap& m) { asm volatile("prefetch.tensormap [%0];" ::"l"(&m) : "memory"); }
// one thread of a converged warp, the same one each time
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}
// whether a barrier's phase has completed, without waiting
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

template <class T>
__device__ __forceinline__ void finish_any(int act, const float* slot, int lane, const float (&bias)[4], const Four<T> (&extra)[4], int extra_mode, T* at,
                                           int64_t pitch, int rows, int left, int vector) {
    switch (act) {
        case MXQ_ACT_RELU: finish<MXQ_ACT_RELU>(slot, lane, bias, extra, extra_mode, at, pitch, rows, left, vector); break;
        case MXQ_ACT_GELU: finish<MXQ_ACT_GELU>(slot, lane, bias, extra, extra_mode, at, pitch, rows, left, vector); break;
        case MXQ_ACT_GELU_TANH: finish<MXQ_ACT_GELU_TANH>(slot, lane, bias, extra, extra_mode, at, pitch, rows, left, vector); break;
        case MXQ_ACT_SILU: finish<MXQ_ACT_SILU>(slot, lane, bias, extra, extra_mode, at, pitch, rows, left, vector); break;
        default: finish<MXQ_ACT_NONE>(slot, lane, bias, extra, extra_mode, at, pitch, rows, left, vector); break;
    }
}
// zeros into the rows before the first group (begin) and behind the last one (end), by `threads` threads of every CTA
template <class T>
__device__ __forceinline__ void zero_rows_outside(T* out, int begin, int end, int rows, int N, int thread, int threads) {
    const int64_t before = (int64_t)begin * N, rest = before + (int64_t)(rows - end) * N;
    for (int64_t i = (int64_t)blockIdx.x * threads + thread; i < rest; i += (int64_t)gridDim.x * threads)
        narrow(0.0f, out[i < before ? i : i - before + (int64_t)end * N]);
}

// 1.0 (two of them for the 16-bit types) as a word
template <class KIn> __device__ __forceinline__ constexpr uint32_t one_bits() {
    return KIn::size == 4 ? 0x3F800000u : std::is_same<KIn, KBF16>::value ? 0x3F803F80u : 0x3C003C00u;
}

// Codes of a narrower element format, one per byte, as the E4M3 bytes of the same values (exact).
template <class F> __device__ __forceinline__ uint32_t widen_codes4(uint32_t w) {
    if constexpr (F{}.eb() == 2 && F{}.fb() == 1) {
        // the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 looked up by the three low bits
        const uint32_t pick = (w & 0x7u) | ((w >> 4) & 0x70u) | ((w >> 8) & 0x700u) | ((w >> 12) & 0x7000u);
        return __byte_perm(0x3C383000u, 0x4C484440u, pick) | ((w & 0x08080808u) << 4);
    } else {
        uint32_t lo, hi;
        if constexpr (F{}.eb() == 2) {
            asm("cvt.rn.f16x2.e2m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
            asm("cvt.rn.f16x2.e2m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
        } else {
            asm("cvt.rn.f16x2.e3m2x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
            asm("cvt.rn.f16x2.e3m2x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
        }
        uint16_t a, b;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(a) : "r"(lo));
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(b) : "r"(hi));
        return (uint32_t)a | ((uint32_t)b << 16);
    }
}

// Quantising E (8 or 16) elements of a 32-element block per lane, as they lie in memory (the 32 / E lanes of the block are neighbours),
// in four steps, so that a kernel with several blocks per lane can derive each block's header on one lane only.
// Range of the lane's magnitudes: bf16 -- packed pairs of the largest and the smallest, else fp32 bits.
template <class KIn, int E> __device__ __forceinline__ void part_range(const uint32_t (&raw)[E * KIn::size / 4], uint32_t& hi, uint32_t& lo) {
    if constexpr (std::is_same<KIn, KBF16>::value) {
#pragma unroll
        for (int i = 0; i < E / 8; ++i) {
            const Pack<16> p{{raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]}};
            uint32_t h, l;
            bf16_abs_range(p, h, l);
            hi = i == 0 ? h : bf2_bits(__hmax2_nan(bf2(hi), bf2(h)));
            lo = i == 0 ? l : bf2_bits(__hmin2(bf2(lo), bf2(l)));
        }
    } else {
        hi = 0u;
        lo = ~0u;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t m = (KIn::size == 4 ? raw[i * KIn::size / 4] : KIn::to_bits(i & 1 ? raw[i >> 1] >> 16 : raw[i >> 1] & 0xFFFFu)) & 0x7FFFFFFFu;
            hi = max(hi, m);
            lo = min(lo, m);
        }
    }
}
// the block's largest magnitude, on all its lanes
template <class KIn, int E> __device__ __forceinline__ uint32_t part_reduce(uint32_t hi) {
#pragma unroll
    for (int d = 1; d < 32 / E; d <<= 1) {
        const uint32_t other = __shfl_xor_sync(~0u, hi, d);
        if constexpr (std::is_same<KIn, KBF16>::value) hi = bf2_bits(__hmax2_nan(bf2(hi), bf2(other)));
        else hi = max(hi, other);
    }
    return hi;
}
// the block's header (2^-se, scale byte, whether it holds Inf / NaN) and a second word: what the packed bf16 quantisers share, else the
// bound of the short form
template <class KIn, class F> __device__ __forceinline__ uint2 part_header(uint32_t hi) {
    const F f{};
    if constexpr (std::is_same<KIn, KBF16>::value) {
        const uint32_t header = block_header_bf16(bf16x2_max_bits(hi), f);
        return make_uint2(header, bf16_block_word<F>(header));
    } else {
        const uint32_t header = block_header(hi, f);
        uint32_t bound = 0u;
        if constexpr (PkFmt<F>::RARE_SUBRANGE) bound = short_form_limit_bits<F>(header);
        return make_uint2(header, bound);
    }
}
// The tensor cores' codes, and the block's scale byte as the result.  bf16 inputs take the packed quantisers, the 8-bit element formats
// their short form where no element of the warp lies below its block's normal range (so lanes without a row should hold
// ones, not zeros).  A block with a code that the hardware reads as Inf / NaN becomes (scale + 1, elements / 2).
// OUT: 0 = E4M3 bytes, 1 = E5M2 bytes, 5 = E2M1 nibbles.
template <class KIn, class F, int OUT, int E>
__device__ __forceinline__ uint32_t part_encode(const uint32_t (&raw)[E * KIn::size / 4], uint32_t lo, uint2 header, uint32_t (&codes)[OUT == 5 ? E / 8 : E / 4]) {
    const F f{};
    uint32_t o[E / 4], sbyte = (header.x >> 8) & 0xFFu;
    const bool special = header.x & 1u;
    if constexpr (std::is_same<KIn, KBF16>::value) {
#pragma unroll
        for (int i = 0; i < E / 8; ++i) {
            const Pack<16> p{{raw[4 * i], raw[4 * i + 1], raw[4 * i + 2], raw[4 * i + 3]}};
            bf16_quantise_access<F, false>(p, header.y, lo, header.x, 0u, o + 2 * i);
        }
    } else {
        uint32_t b[E];
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] = KIn::size == 4 ? raw[i * KIn::size / 4] : KIn::to_bits(i & 1 ? raw[i >> 1] >> 16 : raw[i >> 1] & 0xFFFFu);
        const float inv = __uint_as_float(header.x & 0x7F800000u);
        bool short_form = false;
        if constexpr (PkFmt<F>::RARE_SUBRANGE) short_form = !__any_sync(~0u, lo < header.y);
        if (short_form) {
            if constexpr (PkFmt<F>::RARE_SUBRANGE) {
#pragma unroll
                for (int i = 0; i < E / 4; ++i) o[i] = f32_codes4_normal(b + 4 * i, inv, f);
            }
        } else {
            uint32_t qb[E], mag[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                qb[i] = mx_quotient_bits(b[i], inv);
                mag[i] = (uint32_t)encode_mag_fp(qb[i], f);
            }
#pragma unroll
            for (int i = 0; i < E / 4; ++i) o[i] = pack4_codes(mag + 4 * i, qb + 4 * i, f);
        }
    }
    if constexpr (F{}.eb() >= 4) {
        // carry out of the magnitude byte: a code the hardware reads as Inf / NaN
        constexpr uint32_t probe = F{}.eb() == 4 ? 0x01010101u : 0x04040404u;
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) bad |= ((o[i] & 0x7F7F7F7Fu) + probe) & 0x80808080u;
#pragma unroll
        for (int d = 1; d < 32 / E; d <<= 1) bad |= __shfl_xor_sync(~0u, bad, d);
        if (bad != 0u) {
#pragma unroll
            for (int i = 0; i < E / 4; ++i) o[i] = halve_codes4<F{}.fb()>(o[i]);
            sbyte += sbyte < 255u ? 1u : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        if (special) o[i] = 0u;
        if constexpr (OUT == 5) {
            uint32_t t = o[i] & 0x0F0F0F0Fu;                              // element 2i in the low nibble of byte i
            t |= t >> 4;
            t = (t & 0xFFu) | ((t >> 8) & 0xFF00u);
            if (i % 2 == 0) codes[i / 2] = t; else codes[i / 2] |= t << 16;
        } else if constexpr (F{}.eb() >= 4) {
            codes[i] = o[i];
        } else {
            codes[i] = widen_codes4<F>(o[i]);
        }
    }
    return special ? 255u : sbyte;                                       // 255 is NaN to the tensor cores, whatever the codes
}
// all four steps; all lanes of the warp take part
template <class KIn, class F, int OUT, int E>
__device__ __forceinline__ uint32_t quantise_part(const uint32_t (&raw)[E * KIn::size / 4], uint32_t (&codes)[OUT == 5 ? E / 8 : E / 4]) {
    uint32_t hi, lo;
    part_range<KIn, E>(raw, hi, lo);
    return part_encode<KIn, F, OUT, E>(raw, lo, part_header<KIn, F>(part_reduce<KIn, E>(hi)), codes);
}

// fn(F, the operand's format) for a built-in round-to-nearest format; `nibbles`: E2M1 stays packed in four bits
template <class Fn> static void with_row_format(int eb, int fb, bool nibbles, Fn&& fn) {
    with_preset(eb, fb, 1, MXQ_RN, [&](auto fmt) {
        using F = decltype(fmt);
        if constexpr (F{}.eb() == 5) fn(fmt, std::integral_constant<int, 1>{});
        else if constexpr (F{}.eb() == 2 && F{}.fb() == 1) { if (nibbles) fn(fmt, std::integral_constant<int, 5>{}); else fn(fmt, std::integral_constant<int, 0>{}); }
        else fn(fmt, std::integral_constant<int, 0>{});
    });
}

// The tensor-core instructions for one CTA or for a pair (CTAS = 2: the leader issues, both CTAs' shared and tensor memory take part).
template <int CTAS> __device__ __forceinline__ void tc_alloc(uint32_t slot, int columns) {
    if constexpr (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS> __device__ __forceinline__ void tc_dealloc(uint32_t tmem, int columns) {
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
template <int CTAS> __device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CTAS == 1) tmem_cp_32x128b(taddr, desc);
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int CTAS, bool MXF4>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CTAS == 1 && MXF4) mma_mxf4(d, a, b, idesc, sfa, sfb, accumulate);
    else if constexpr (CTAS == 1) mma_mxf8f6f4(d, a, b, idesc, sfa, sfb, accumulate);
    else if constexpr (MXF4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
}
// arrives on the barrier at this address of every CTA of the pair once the products so far are done
template <int CTAS> __device__ __forceinline__ void tc_commit(uint32_t bar) {
    if constexpr (CTAS == 1) mma_commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// tiled load into this CTA's shared memory that completes a barrier of either CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Clusters: an address in another CTA's shared memory, arrival on another CTA's barrier (behind this thread's accesses), a barrier of
// all threads, and bounded waits for what other CTAs complete.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void arrive_at(uint32_t bar, int rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(bar, (uint32_t)rank)) : "memory");
}
// The same behind reads of tensor memory that products of another CTA's thread will overwrite: those are ordered by
// tcgen05.fence::before_thread_sync here, ::after_thread_sync there and a relaxed arrival of cluster scope between them.  A release would
// wait for the thread's stores as well (8192 rows over 32 experts of 2048 x 2048, 4-bit pairs: 63 -> 68 us).
__device__ __forceinline__ void arrive_after_tensor_reads(uint32_t bar, int rank) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(bar, (uint32_t)rank)) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool mbar_test_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, int* status, int code) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (i > 64) __nanosleep(32);
    }
    if (status) *reinterpret_cast<volatile int*>(status) = code;
    return false;
}

// where a unit of work lies: features [f0, f0 + FEATURES) of group g for rows [row, row + rows)
struct Unit {
    int g, f0, ftile, row, rows;
    int begin, tile;             // first row of the group, row tile within it
    __device__ __forceinline__ uint32_t padded() const { return (uint32_t)(rows + 15) & ~15u; }
};

// Position in a ring of STAGES stages, and the parity of its barriers' current phase.
template <int STAGES> struct RingAt {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void step() { if (++s == STAGES) { s = 0; phase ^= 1u; } }
    __device__ __forceinline__ void step(int n) { for (s += n; s >= STAGES; s -= STAGES) phase ^= 1u; }
};

// Rows per tile of a group of n rows cut into tt = ceil(n / width) tiles: equal, a multiple of 16, at most `width`; the last tile is never empty.
__device__ __forceinline__ int tile_rows(int n, int tt) { return tt == 1 ? (n + 15) & ~15 : ((n + tt - 1) / tt + 15) & ~15; }

// The group table (tile counts summed over the groups, first rows) and the walk over the units of one CTA.  Called by whole warps.
struct Walk {
    const int *tiles, *first;
    int g, groups, ftiles, total;
    __device__ __forceinline__ Walk(const int* t, const int* f, int groups_, int ftiles_)
        : tiles(t), first(f), g(0), groups(groups_), ftiles(ftiles_), total(t[groups_] * ftiles_) {}
    __device__ __forceinline__ Unit at(int u, int features) {
        // units are visited in rising order: the first group from g on that ends behind u, 32 groups a step
        if (groups > 1) {
            for (;; g += 32) {
                const int i = g + (threadIdx.x & 31);
                const uint32_t behind = __ballot_sync(~0u, i < groups && u < tiles[min(i, groups - 1) + 1] * ftiles);
                if (behind != 0u) { g += __ffs(behind) - 1; break; }
            }
        }
        const int tt = tiles[g + 1] - tiles[g], begin = first[g], n = first[g + 1] - begin, local = u - tiles[g] * ftiles;
        int ti = 0, fi = local;
        if (tt > 1) tile_coords(local, tt, ftiles, ti, fi);
        const int w = tile_rows(n, tt);
        return Unit{g, fi * features, fi, begin + ti * w, min(w, n - ti * w), begin, ti};
    }
};

// The rows of a call and how they are grouped.
struct Groups {
    const void* offsets;         // [groups + 1], or null: one group of all rows
    int offsets64, rows, groups;
    int width;                   // rows per tile at most (a multiple of 16)
    __device__ __forceinline__ int offset(int i) const {
        if (offsets == nullptr) return i == 0 ? 0 : rows;
        const int64_t v = offsets64 ? reinterpret_cast<const long long*>(offsets)[i] : (int64_t)reinterpret_cast<const int*>(offsets)[i];
        return (int)min(max(v, (int64_t)0), (int64_t)rows);
    }
};

// The group table, by the whole CTA: first[i] = the largest of offsets[0 .. i] (offsets that fall back leave an empty group and never
// an overlap), tiles[i] = row tiles of the groups before i.  The offsets are loaded by all threads at once, one warp sums.
__device__ __forceinline__ void build_table(const Groups& g, int* tiles, int* first) {
    for (int i = threadIdx.x; i <= g.groups; i += blockDim.x) first[i] = g.offset(i);
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int high = 0, sum = 0;
        for (int base = 0; base <= g.groups; base += 32) {
            const int i = base + lane;
            int v = i <= g.groups ? first[i] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(~0u, v, o); if (lane >= o) v = max(v, up); }
            v = max(v, high);
            const int before = __shfl_up_sync(~0u, v, 1);
            // rows of group i - 1, which the running sum at i counts
            int t = (i == 0 || i > g.groups) ? 0 : ((v - (lane == 0 ? high : before)) + g.width - 1) / g.width;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(~0u, t, o); if (lane >= o) t += up; }
            t += sum;
            if (i <= g.groups) { first[i] = v; tiles[i] = t; }
            high = __shfl_sync(~0u, v, 31);
            sum = __shfl_sync(~0u, t, 31);
        }
    }
    __syncthreads();
}

// Where the scales of one row lie: its tile's slot and its row in the tile.
struct Place {
    int slot, r;
    __device__ __forceinline__ Place() : slot(-1), r(0) {}
    __device__ __forceinline__ Place(const Groups& g, int group, int begin, int end, int row) {
        const int n = end - begin, w = tile_rows(n, (n + g.width - 1) / g.width), t = (row - begin) / w;
        slot = begin / g.width + group + t;
        r = row - begin - t * w;
    }
    // byte of K block kb: chunk r / 128 of its 128-element step, (r % 32) * 16 + (r % 128 / 32) * 4 + kb % 4 within
    __device__ __forceinline__ int64_t at(int kb, int KT128, int chunks) const {
        return (((int64_t)slot * KT128 + (kb >> 2)) * chunks + (r >> 7)) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + (kb & 3);
    }
};

// The whole CTA: place of one row, slot -1 for a row of no group.  The group is the first whose end lies behind the row (in the
// running maximum of the offsets, that is the first offset behind it), its begin the largest offset up to there.
__device__ __forceinline__ Place find_row(const Groups& g, int row, int* s_two) {
    if (g.offsets == nullptr) return Place(g, 0, 0, g.rows, row);
    if (threadIdx.x == 0) { s_two[0] = g.groups; s_two[1] = 0; }
    __syncthreads();
    int group = g.groups;
    for (int e = threadIdx.x; e < g.groups && group == g.groups; e += blockDim.x) if (g.offset(e + 1) > row) group = e;
    group = __reduce_min_sync(~0u, group);
    if ((threadIdx.x & 31) == 0) atomicMin(&s_two[0], group);
    __syncthreads();
    group = s_two[0];
    if (group == g.groups) return Place();
    int begin = 0;
    for (int e = threadIdx.x; e <= group; e += blockDim.x) begin = max(begin, g.offset(e));
    begin = __reduce_max_sync(~0u, begin);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_two[1], begin);
    __syncthreads();
    begin = s_two[1];
    return begin > row ? Place() : Place(g, group, begin, g.offset(group + 1), row);
}

struct Params {
    const uint8_t* w;            // packed weights (WeightTile blocks)
    int64_t w_group;             // bytes per group
    const uint8_t* x_sf;         // row scales
    void* out;
    const void* bias;            // [groups, N] or null
    const void* extra;           // [rows, N] or null
    Groups rows;
    int N, K;
    int act, extra_mode;
    int zero_rest;               // write zeros into the rows that belong to no group
    int vector;                  // out, extra and their rows are aligned to four elements
    uint32_t idesc;              // instruction descriptor without the width
    int* status;
};

// units of work at most: every group may end in a partial tile; what the groups leave is known on the device only
static int64_t most_units(const Groups& g, int64_t N, int features) {
    return (int64_t)(g.rows / g.width + (g.groups < g.rows ? g.groups : g.rows)) * ((N + features - 1) / features);
}

// mxq_grouped_decode.cu: rows that fit tiles of decode_rows(); x on 16 bytes, a built-in round-to-nearest format
int decode_rows();
int launch_decode(const Params& p, int dt, const void* x, const void* row_index, int index64, int64_t rows_in, int eb, int fb, bool nibbles,
                  cudaStream_t st);

template <class... KArgs, class... Args>
static int launch_after(void (*kernel)(KArgs...), unsigned grid, unsigned block, unsigned smem, unsigned cluster, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    if (e != cudaSuccess) { set_last_cuda_error(e); return MXQ_ELAUNCH; }
    return check_launch();
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
// box of `box` lines of 128 bytes, as they lie in memory
static bool make_line_map(CUtensorMap* map, const void* lines, int64_t n, int box) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {128, (cuuint64_t)n};
    const cuuint64_t strides[1] = {128};
    const cuuint32_t boxes[2] = {128, (cuuint32_t)box};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(lines), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace grouped
}  // namespace mxq
