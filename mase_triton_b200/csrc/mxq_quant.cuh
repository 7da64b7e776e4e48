// Element quantisers shared by the kernels that write MXFP codes: two bf16 elements per 32-bit word on the packed bf16 units, the
// short forms for the 8-bit element formats, and the halving of codes that the tensor cores' format lacks.
#pragma once
#include "mxq_device.cuh"

namespace mxq {

// ------------------------------------------------------------------------------------------------
// MXFP4 (E2M1) elements of bf16 inputs, two elements per 32-bit word on the packed bf16 units.
// The quotient q = |x| * 2^-se is exact in bf16 for a power-of-two factor (below 2^-126 it only has
// to stay below 0.625), and q < 8 for a finite block.  Per word:
//   * q >= 1: the 7-bit mantissa, tagged with exponent 0, plus 63.0 is 64 + (m - 1) rounded half to
//     even to a multiple of 0.5, so the sum's bits are those of 64.0 plus fr in {0, 1, 2}; fr << 6
//     OR-ed under q's own exponent field is the quantised quotient in bf16 (fr = 2 lands on the
//     exponent's low bit: the reference's OR-merge, minifloat/fake.py:70, carry lost for odd fields);
//     the code is that pattern shifted down, re-biased with one XOR;
//   * q < 1: the single subnormal binade (:56-60) leaves code 1 (0.5) above 0.625 and zero below.
// An element is kept (else it is +0) when it is not a flushed input and its fp32 quotient does not
// round to zero: |x| > max(2^(se-150), largest subnormal), one packed comparison against a
// per-block constant; the sign bit rides along with the kept ones.
// This is ~8 integer-pipe instructions per element instead of ~13 for the generic codec.
// ------------------------------------------------------------------------------------------------
struct E2M1Block {
    uint32_t inv2;    // 2^-se in both halves
    uint32_t sf2;     // 2^se in both halves (fused form)
    uint32_t ts2;     // keep threshold in both halves
};

__device__ __forceinline__ E2M1Block e2m1_block(uint32_t h) {
    E2M1Block b;
    const uint32_t sb = (h >> 8) & 0xFFu;
    b.inv2 = ((h >> 16) & 0x7F80u) * 0x10001u;
    b.sf2 = (sb == 0u ? 0x0040u : (sb << 7)) * 0x10001u;
    b.ts2 = (uint32_t)max(((int)sb - 150) * 128, 0x7F) * 0x10001u;
    return b;
}

__device__ __forceinline__ __nv_bfloat162 bf2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
__device__ __forceinline__ uint32_t bf2_bits(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

// one 16-byte access of a lane (8 bf16 inputs) of a finite block -> 8 code bytes or 8 bf16 results
template <bool VALUES>
__device__ __forceinline__ void e2m1_bf16_quantise(const Pack<16>& p, const E2M1Block& b, uint32_t* out) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = p.w[i];
        const uint32_t aw = w & 0x7FFF7FFFu;
        const __nv_bfloat162 q = __hmul2(bf2(aw), bf2(b.inv2));
        const uint32_t qb = bf2_bits(q);
        const uint32_t keep = __hgt2_mask(bf2(aw), bf2(b.ts2));
        // normal range: rounded mantissa field under q's exponent field
        const uint32_t sum = bf2_bits(__hadd2(bf2((qb & 0x007F007Fu) | 0x3F803F80u), bf2(0x427C427Cu)));      // + 63.0
        const uint32_t z = sum * (uint32_t)rt_k(9) - 0x42804280u * 64u;        // (sum - bits(64.0)) << 6 per half, as one multiply-add
        const uint32_t y = (qb & 0x7F807F80u) | z;
        const uint32_t lt1 = __hlt2_mask(q, bf2(0x3F803F80u));                  // q < 1
        const uint32_t gt = __hgt2_mask(q, bf2(0x3F203F20u));                   // q > 0.625
        if constexpr (VALUES) {
            const uint32_t v = (lt1 & gt & 0x3F003F00u) | (~lt1 & y);            // 0.5 / 0 below 1, else the quantised quotient
            const uint32_t o = bf2_bits(__hmul2(bf2(v), bf2(b.sf2)));
            r[i] = ((o & 0x7FFF7FFFu) | (w & 0x80008000u)) & keep;
        } else {
            const uint32_t cn = ((y >> 6) ^ 0x00040004u) & 0x00070007u;          // (E << 1 | fr) - 252, modulo 8
            const uint32_t c = (lt1 & gt & 0x00010001u) | (~lt1 & cn);
            r[i] = (c | ((w >> 12) & 0x00080008u)) & keep;
        }
    }
    if constexpr (VALUES) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = r[i];
    } else {
        out[0] = __byte_perm(r[0], r[1], 0x6420);
        out[1] = __byte_perm(r[2], r[3], 0x6420);
    }
}

// ------------------------------------------------------------------------------------------------
// The same idea for the other element formats (E4M3, E5M2, E2M3, E3M2) of bf16 inputs: two elements
// per 32-bit word on the packed bf16 units.  For a quotient q = |x| * 2^-se (exact in bf16):
//   * normal range (biased exponent >= 1): the 7-bit mantissa, tagged with exponent 0, plus 2^(7-fb)
//     rounds half to even to fb fraction bits, so the sum's low bits are 2^fb + fr with fr in
//     [0, 2^fb]; the code is q's exponent field, re-biased by flipping its bit eb-1 (127 - bias is
//     2^(eb-1) modulo 2^eb), with fr OR-ed in -- fr = 2^fb lands on the exponent's low bit, which is the
//     reference's OR-merge with its lost carry (minifloat/fake.py:70-75); the dequantised value is fr
//     OR-ed under q's own exponent field;
//   * below 2^(1-bias): the single subnormal binade (fake.py:56-60) encodes as (fr | 2^fb) >> 1 unless
//     fr is zero, anything below 2^-bias as zero.  For the 8-bit formats such elements are rare and the lanes of a
//     warp skip this part together when none of them has one;
//   * an element is kept (else it is +0) when it is not a flushed input and its fp32 quotient does not
//     round to zero: one packed comparison against a per-block threshold; the sign rides along.
// A bf16 input has 7 mantissa bits, so the reference's cut to 15 bits (fake.py:45) changes nothing.
// ------------------------------------------------------------------------------------------------
template <class F> struct PkFmt {
    static constexpr int EB = F{}.eb(), FB = F{}.fb();
    static constexpr int BIAS = (1 << (EB - 1)) - 1;
    static constexpr uint32_t rep(uint32_t half) { return half * 0x10001u; }
    static constexpr uint32_t ROUND_C = rep((uint32_t)(127 + 7 - FB) << 7);                      // 2^(7-fb)
    static constexpr uint32_t SUM_BASE = rep(((uint32_t)(127 + 7 - FB) << 7) + (1u << FB));      // bits of 2^(7-fb) with mantissa field 2^fb
    static constexpr uint32_t EXP_FLIP = rep((1u << (EB - 1)) << FB);
    static constexpr uint32_t MAG_MASK = rep((1u << (EB + FB)) - 1u);
    static constexpr uint32_t EXP_MASK = rep(((1u << EB) - 1u) << FB);
    static constexpr uint32_t FR_ONE = rep(1u << FB);
    static constexpr uint32_t SUB_MASK = rep((2u << FB) - 1u);
    static constexpr uint32_t SIGN_BIT = rep(1u << (EB + FB));
    static constexpr uint32_t NORMAL_MIN = rep((uint32_t)(128 - BIAS) << 7);                     // 2^(1-bias)
    static constexpr uint32_t BINADE_MIN = rep((uint32_t)(127 - BIAS) << 7);                     // 2^-bias
    static constexpr uint32_t REBIAS = rep((uint32_t)(254 - BIAS) << 7);                         // 2^(127-bias)
    static constexpr bool RARE_SUBRANGE = EB >= 4;       // block maximum >= 2^(emax-bias): elements 2^14 (E4M3) / 2^29 (E5M2) below it
};

// one 16-byte access of a lane (8 bf16 inputs) of a finite block.
// VALUES: 8 bf16 results in out[0..4); else 8 magnitude+sign code bytes in out[0..2)
template <class F, bool VALUES>
__device__ __forceinline__ void pk_bf16_quantise(const Pack<16>& p, const E2M1Block& b, uint32_t* out) {
    using P = PkFmt<F>;
    uint32_t qb[4], fr[4], res[4];
    uint32_t any_sub = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t aw = p.w[i] & 0x7FFF7FFFu;
        qb[i] = bf2_bits(__hmul2(bf2(aw), bf2(b.inv2)));
        const uint32_t sum = bf2_bits(__hadd2(bf2((qb[i] & 0x007F007Fu) | 0x3F803F80u), bf2(P::ROUND_C)));
        fr[i] = sum - P::SUM_BASE;                                           // 0 .. 2^fb in each half
        if constexpr (VALUES) res[i] = (qb[i] & 0x7F807F80u) | (fr[i] << (7 - P::FB));
        else res[i] = (((qb[i] >> (7 - P::FB)) ^ P::EXP_FLIP) & P::EXP_MASK) | fr[i];
        any_sub |= __hlt2_mask(bf2(qb[i]), bf2(P::NORMAL_MIN));
    }
    if (!P::RARE_SUBRANGE || __any_sync(__activemask(), any_sub != 0u)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lt = __hlt2_mask(bf2(qb[i]), bf2(P::NORMAL_MIN));
            const uint32_t ge = __hge2_mask(bf2(qb[i]), bf2(P::BINADE_MIN));
            // (fr | 2^fb) >> 1 when the rounded mantissa field is not zero (fake.py:58), zero otherwise and below the binade
            const uint32_t nz = (((fr[i] + 0x7FFF7FFFu) >> 15) & 0x00010001u) * 0xFFFFu;
            const uint32_t sub = ((fr[i] | P::FR_ONE) >> 1) & P::SUB_MASK & ge & nz;
            if constexpr (VALUES) {
                // sub * 2^(1-bias-fb): the field placed at the top of a bf16 mantissa is sub * 2^(-fb-126)
                const uint32_t v = bf2_bits(__hmul2(bf2(sub << (7 - P::FB)), bf2(P::REBIAS)));
                res[i] = (lt & v) | (~lt & res[i]);
            } else {
                res[i] = (lt & sub) | (~lt & res[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = p.w[i];
        const uint32_t keep = __hgt2_mask(bf2(w & 0x7FFF7FFFu), bf2(b.ts2));
        if constexpr (VALUES) {
            const uint32_t o = bf2_bits(__hmul2(bf2(res[i]), bf2(b.sf2)));
            res[i] = ((o & 0x7FFF7FFFu) | (w & 0x80008000u)) & keep;
        } else {
            res[i] = (res[i] | ((w >> (15 - P::EB - P::FB)) & P::SIGN_BIT)) & keep;
        }
    }
    if constexpr (VALUES) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = res[i];
    } else {
        out[0] = __byte_perm(res[0], res[1], 0x6420);
        out[1] = __byte_perm(res[2], res[3], 0x6420);
    }
}

// ------------------------------------------------------------------------------------------------
// bf16 inputs: what the lanes of a block share, and the short form of the quantiser for the 8-bit formats.
//   * every lane keeps the packed maximum AND minimum of its eight |x| (NaN wins the maximum); the maxima are
//     reduced over the block's lanes as packed pairs, the two halves are only compared on the lane that derives the header;
//   * that lane also derives the packed constants the block's lanes need and hands them over in one word:
//     2^-se and a second bf16 threshold (its own per format, see bf16_block_word);
//   * E4M3 / E5M2: when every |x| of the lanes that vote together is at least 2^(1-bias+se) -- no element in the
//     sub-range, none flushed or rounding to zero, which is nearly always so for these formats -- the code is
//     built from the SIGNED quotient with no per-element case analysis: exponent field and rounded fraction
//     OR-ed per word, the re-bias (one XOR) and the sign bits (one byte gather) applied to four packed codes
//     at a time.  Otherwise the lanes take pk_bf16_quantise, which handles every case.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bf16_abs_range(const Pack<16>& p, uint32_t& mx2, uint32_t& mn2) {
    const __nv_bfloat162 a0 = __habs2(bf2(p.w[0])), a1 = __habs2(bf2(p.w[1])), a2 = __habs2(bf2(p.w[2])), a3 = __habs2(bf2(p.w[3]));
    mx2 = bf2_bits(__hmax2_nan(__hmax2_nan(a0, a1), __hmax2_nan(a2, a3)));
    mn2 = bf2_bits(__hmin2(__hmin2(a0, a1), __hmin2(a2, a3)));
}

// fp32 bits of the larger half of a packed pair of bf16 magnitudes; NaN wins (as 15-bit patterns the magnitudes
// order like integers, NaN above Inf above every finite value)
__device__ __forceinline__ uint32_t bf16x2_max_bits(uint32_t m2) {
    return max(m2 & 0xFFFFu, m2 >> 16) << 16;
}

// block_header for the maximum of bf16 inputs (fp32 bits with 16 zero low bits): such a maximum is never among the
// last floats below a power of two, so the round-up of the reference's log2 (shared_exponent) cannot apply and the
// shared exponent is the exponent field minus the format's largest exponent
template <class F>
__device__ __forceinline__ uint32_t block_header_bf16(uint32_t amax_bits, const F& f) {
    const int emax_b = fmt_emax(f) - fmt_bias(f);
    const uint32_t E = amax_bits >> 23;
    const uint32_t special = E == 255u ? 1u : 0u;
    const int se = max((int)E - 127 - emax_b, -127);
    const uint32_t sbyte = E == 0u ? 0u : (special ? 255u : (uint32_t)(se + 127));
    const uint32_t inv_field = (E == 0u || special) ? 127u : (uint32_t)(127 - se);
    return (inv_field << 23) | (sbyte << 8) | special;
}

// Low half: bf16 bits of 2^-se.  High half, by format: E2M1 -- the keep threshold (e2m1_block's ts2); E4M3 / E5M2 --
// 2^(1-bias+se), the smallest |x| of the short form (+Inf, i.e. never, for blocks so small that flushed inputs
// could lie above it); others: unused.  Bit 31: the block holds Inf / NaN.
template <class F>
__device__ __forceinline__ uint32_t bf16_block_word(uint32_t hdr) {
    const int sb = (int)((hdr >> 8) & 0xFFu);
    uint32_t second = 0u;
    if constexpr (F{}.eb() == 2 && F{}.fb() == 1) {
        second = (uint32_t)max((sb - 150) * 128, 0x7F);
    } else if constexpr (PkFmt<F>::RARE_SUBRANGE) {
        const int e = sb + 1 - PkFmt<F>::BIAS;
        second = e >= 2 ? (uint32_t)e << 7 : 0x7F80u;
    }
    return ((hdr >> 16) & 0x7F80u) | (second << 16) | (hdr << 31);
}

// short form (see above): 8 bf16 inputs of a lane -> 8 code bytes (out[0..2)) or 8 bf16 results (out[0..4))
template <class F, bool VALUES>
__device__ __forceinline__ void pk_bf16_quantise_normal(const Pack<16>& p, uint32_t inv2, uint32_t sf2, uint32_t* out) {
    using P = PkFmt<F>;
    static_assert(P::EB + P::FB == 7, "the sign gather assumes 8-bit codes");
    uint32_t qb[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        qb[i] = bf2_bits(__hmul2(bf2(p.w[i]), bf2(inv2)));                  // signed quotient
        const uint32_t sum = bf2_bits(__hadd2(bf2((qb[i] & 0x007F007Fu) | 0x3F803F80u), bf2(P::ROUND_C)));
        if constexpr (VALUES) {
            // (sum - SUM_BASE) << (7 - fb) as one multiply-add; OR-ed under the quotient's sign and exponent, times 2^se
            const uint32_t z = sum * (uint32_t)rt_k(P::FB == 3 ? 10 : 11) - P::SUM_BASE * (1u << (7 - P::FB));
            r[i] = bf2_bits(__hmul2(bf2((qb[i] & 0xFF80FF80u) | z), bf2(sf2)));
        } else {
            const uint32_t fr = sum * (uint32_t)rt_k(0) - P::SUM_BASE;       // 0 .. 2^fb in each half
            r[i] = ((qb[i] >> (7 - P::FB)) & P::EXP_MASK) | fr;             // exponent field not re-biased yet
        }
    }
    if constexpr (VALUES) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = r[i];
    } else {
        constexpr uint32_t FLIP4 = ((1u << (P::EB - 1)) << P::FB) * 0x01010101u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t mag4 = __byte_perm(r[2 * i], r[2 * i + 1], 0x6420) ^ FLIP4;
            const uint32_t sgn4 = __byte_perm(qb[2 * i], qb[2 * i + 1], 0x7531);        // the halves' upper bytes: sign on top
            out[i] = mag4 | (sgn4 & 0x80808080u);
        }
    }
}

// One 16-byte access of a lane of a finite block, every format: picks the short form where it applies.
// `w2` is the block word, `mn2` this lane's packed minimum, `h` the block header (only read on the full path).
template <class F, bool VALUES>
__device__ __forceinline__ void bf16_quantise_access(const Pack<16>& p, uint32_t w2, uint32_t mn2, uint32_t h, uint32_t sf2, uint32_t* out) {
    const uint32_t inv2 = __byte_perm(w2, 0u, 0x1010);
    const uint32_t second2 = __byte_perm(w2, 0u, 0x3232);
    if constexpr (F{}.eb() == 2 && F{}.fb() == 1) {
        // (a vote that skips the keep threshold when no lane holds an element at or below it was measured: no gain)
        E2M1Block b;
        b.inv2 = inv2; b.sf2 = sf2; b.ts2 = second2;
        e2m1_bf16_quantise<VALUES>(p, b, out);
    } else if constexpr (PkFmt<F>::RARE_SUBRANGE) {
        const bool any_below = __any_sync(__activemask(), __hlt2_mask(bf2(mn2), bf2(second2)) != 0u);
        if (!any_below) pk_bf16_quantise_normal<F, VALUES>(p, inv2, sf2, out);
        else pk_bf16_quantise<F, VALUES>(p, e2m1_block(h), out);
    } else {
        pk_bf16_quantise<F, VALUES>(p, e2m1_block(h), out);
    }
}

// fp32 inputs, E4M3 / E5M2 codes: the short form of the element encode, as pk_bf16_quantise_normal.  When every
// |x| of the lanes that vote together is at least 2^(1-bias+se) (`lim`), nothing is flushed, in the sub-range or
// rounding to zero, so four codes are: exponent field (low eb bits, re-biased later) OR rounded fraction per
// element from the SIGNED quotient, packed, re-biased with one XOR, signs gathered from the quotients' top bytes.
template <class F>
__device__ __forceinline__ uint32_t f32_codes4_normal(const uint32_t* x_bits, float inv, const F& f) {
    constexpr int fb = F{}.fb(), eb = F{}.eb();
    constexpr uint32_t cbits = (uint32_t)(127 + 23 - fb) << 23;           // 2^(23-fb)
    uint32_t qb[4], mag[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        qb[i] = __float_as_uint(__fmul_rn(__uint_as_float(x_bits[i]), inv));
        // the reference's cut of the mantissa to 15 bits (minifloat/fake.py:45) commutes with the exact scaling
        const float m = __uint_as_float((qb[i] & 0x007FFF00u) | 0x3F800000u);
        const uint32_t fr = (uint32_t)mad_add((int)__float_as_uint(__fadd_rn(m, __uint_as_float(cbits))), -(int)(cbits + (1u << fb)));
        mag[i] = ((qb[i] >> (23 - fb)) & (((1u << eb) - 1u) << fb)) | fr;
    }
    return pack4_codes(mag, qb, f) ^ (((1u << (eb - 1)) << fb) * 0x01010101u);
}

// per-block bound of the short form as fp32 bits, from the block header (+Inf: never)
template <class F>
__device__ __forceinline__ uint32_t short_form_limit_bits(uint32_t hdr) {
    const int e = (int)((hdr >> 8) & 0xFFu) + 1 - PkFmt<F>::BIAS;
    return (uint32_t)(e >= 2 ? e : 255) << 23;
}

__device__ __forceinline__ float f32x4_absmin(const Pack<16>& p) {
    return fminf(fminf(fabsf(__uint_as_float(p.w[0])), fabsf(__uint_as_float(p.w[1]))),
                 fminf(fabsf(__uint_as_float(p.w[2])), fabsf(__uint_as_float(p.w[3]))));
}

// Four hardware magnitude+sign code bytes of a block that is stored with its scale raised by one: every
// magnitude becomes the code of half the value -- exponent minus one for codes with exponent >= 2, a
// round-half-to-even shift for the two lowest binades -- on all four bytes of the word at once.
template <int FB>
__device__ __forceinline__ uint32_t halve_codes4(uint32_t c) {
    constexpr uint32_t ONE = 0x01010101u;
    const uint32_t mag = c & 0x7F7F7F7Fu;
    // per byte: 0xFF where mag >= 2 << FB (adding 0x80 - (2 << FB) carries into bit 7 exactly then)
    const uint32_t big = (((mag + ONE * (0x80u - (2u << FB))) >> 7) & ONE) * 0xFFu;
    const uint32_t normal = mag - (big & (ONE << FB));                       // no borrow: those bytes are >= 2 << FB
    const uint32_t small = ((mag + ((mag >> 1) & ONE)) >> 1) & 0x7F7F7F7Fu;   // bytes < 2 << FB: no carry out of the byte
    return (big & normal) | (~big & small) | (c & 0x80808080u);
}

}  // namespace mxq
