// The experts' products over a plan (MoeArgs): tiles of up to 64, or 32, of one expert's slots times 256 or 128
// weight rows (half of them of gate and half of up), on v_mfma_f32_32x32x16_f16.
//
// The product is computed transposed, D[slot][row], so that a lane holds one weight row in all of its
// accumulators and a block's scale is one per-lane factor. Work-group: 4 waves, each the tile's slots
// times 64 or 32 rows of its own in tiles of 32 x 32 (gate_up: rows of gate beside the same rows of up, in the
// lane's two row tiles or 16 lanes apart, so the activation stays in the wave). A weight is thus decoded by one
// wave only, and the slots' inputs, four bytes an element where the weights have half to one, are shared by all
// rows. Tiles of at most 32 slots skip the second half.
// - Weights: windows of WB k-blocks move through registers (the next window in flight while this one is
//   multiplied) into the wave's LDS; lane l copies 16-byte pieces of rows 32 (l / 32) .. + 31.
// - Inputs: pairs of k-blocks, f16 (hi and lo), 64 bytes per slot and block, whose 16-byte chunk c (k 8c ..)
//   is at c ^ swz(slot); two buffers, the pair after the next in registers; one barrier per pair.
//
// Scales cost a vector instruction per accumulator and k-block beside 32 cycles of MFMA, so where the
// formats allow they are part of the operand, exactly, and the accumulators run through:
// - MXFP4: 2^(e - 127) scales the E2M1 code in the conversion, exact while every product is a normal f16,
//   which is checked per window (e from 114 to 139). A work-group that finds another e, a zero block's e = 0 too, runs
//   its reduction again and scales each block's f32 sum: 2000 tokens of 32 experts 906 us, and 1827 with one zero block
//   in 4000, which leaves hardly a work-group without.
// - Q4_K, Q5_K: 6-bit scale times 4- or 5-bit weight is an integer below 2048. The super-block's f16 factor
//   d stays out: the accumulators hold the sum over d, and are multiplied by d_before / d_now between two
//   super-blocks (two roundings in 256 elements). The mins are two MFMAs per super-block on the sums of x over
//   its blocks, each sum as three bf16 pieces (exact, and without f16's range).
// - Q6_K: 8-bit scale times 6-bit weight, up to 4096, takes 13 bits: f16 rounds it by at most 1 above 2048, and
//   the part lost, -1, 0 or 1, is multiplied too (by x's high half; the low one's share is 2^-22).
// - Q8_0: f16 scale times 8 bits does not fit, each block's f32 sum is scaled.
#include "common.h"

namespace {

typedef float moe_f32x16 __attribute__((ext_vector_type(16)));

// A row's window in LDS: bytes where they belong but for Q6_K's last piece (bytes 194 .. 209), which goes to
// 208 .. 223. Lanes read 8 bytes of 32 rows at once, so rows are 2 dwords apart modulo the 32 banks times an odd
// number (136, 152, 184, 232 bytes); F16's 16-byte reads want 4. Q5_K with f32 inputs has no room for that
// beside two work-groups per CU.
template <uint32_t TY, int HALVES>
struct MoeTileFmt {
    static constexpr uint32_t WB = TY == 1 ? 2 : TY == 8 ? 4 : 8;
    static constexpr uint32_t S = WB * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
    static constexpr uint32_t NP = (S + 15u) / 16u;       // 16-byte pieces of a row's window
    static constexpr uint32_t RS = TY == 1 ? 144 : TY == 12 ? 152 : TY == 13 ? (HALVES == 2 ? 176 : 184) : TY == 14 ? 232 : 136;
};

// The order of a k-block's 32 inputs, the one in which its weights are cheapest to unpack (the sum does not
// mind): MXFP4 elements j and j + 16 side by side, 4 j's a chunk of 8; K-quants 0 2 1 3 of every four.
__device__ __forceinline__ uint32_t moe_place(uint32_t ty, uint32_t k) {  // where element k is
    if (ty == 39u) {
        const uint32_t j = k & 15u;
        return 8u * (2u * ((j >> 2) & 1u) + (j >> 3)) + 2u * (j & 3u) + (k >> 4);
    }
    if (ty == 12u || ty == 13u || ty == 14u) return (k & ~3u) | ((k & 1u) << 1) | ((k >> 1) & 1u);
    return k;
}

__device__ __forceinline__ uint32_t moe_swz(uint32_t t) { return (t >> 2) & 3u; }

// Every LDS access of this wave is done, and then every wave's. Loads into registers stay in flight.
__device__ __forceinline__ void moe_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ half8_t moe_times(half8_t q, _Float16 f) {
    half8_t r;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const half2_t p = half2_t{q[k], q[k + 1]} * half2_t{f, f};
        r[k] = p[0];
        r[k + 1] = p[1];
    }
    return r;
}
// What f16 lost of q f (exact: the product has 13 bits)
__device__ __forceinline__ half8_t moe_lost(half8_t q, _Float16 f, half8_t product) {
    half8_t r;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const half2_t p = __builtin_elementwise_fma(half2_t{q[k], q[k + 1]}, half2_t{f, f}, half2_t{-product[k], -product[k + 1]});
        r[k] = p[0];
        r[k + 1] = p[1];
    }
    return r;
}

// The 6-bit scale (and min) of block i of a K-quant super-block from its first 16 bytes
__device__ __forceinline__ uint32_t moe_k4_scale(u32x4_t hd, uint32_t i) {
    const uint32_t sh = 8u * (i & 3u);
    return i < 4u ? (hd[1] >> sh) & 63u : ((hd[3] >> sh) & 15u) | (((hd[1] >> (sh + 6u)) & 3u) << 4);
}
__device__ __forceinline__ uint32_t moe_k4_min(u32x4_t hd, uint32_t i) {
    const uint32_t sh = 8u * (i & 3u);
    return i < 4u ? (hd[2] >> sh) & 63u : ((hd[3] >> (sh + 4u)) & 15u) | (((hd[2] >> (sh + 6u)) & 3u) << 4);
}

// The eight bytes at p + OFF, p 8-byte aligned, OFF known at compile time.
__device__ __forceinline__ void moe_get8(uint32_t &d0, uint32_t &d1, const uint8_t *p, uint32_t off) {
    if (off % 8u == 0u) {
        const u32x2_t v = *(const u32x2_t *) (p + off);
        d0 = v[0];
        d1 = v[1];
        return;
    }
    const uint32_t *w = (const uint32_t *) (p + (off & ~3u));
    if (off % 4u == 0u) {
        d0 = w[0];
        d1 = w[1];
        return;
    }
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2];
    d0 = __builtin_amdgcn_alignbyte(w1, w0, off & 3u);
    d1 = __builtin_amdgcn_alignbyte(w2, w1, off & 3u);
}

// The lane's operands of k-block i of a row's window in LDS, slices s = 0, 1, 8 elements each in the order of
// moe_place: f16 integers, times the scale where the format allows. live 0: zeros.
__device__ __forceinline__ half2_t moe_h2(uint32_t bits) { return __builtin_bit_cast(half2_t, bits); }
__device__ __forceinline__ void moe_set(half8_t &w, int k, half2_t p) {
    w[k] = p[0];
    w[k + 1] = p[1];
}
__device__ __forceinline__ void moe_f16_block(half8_t (&w)[2], const uint8_t *row, uint32_t i, uint32_t h, uint32_t live) {
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        u32x4_t v = *(const u32x4_t *) (row + 64u * i + 32u * s + 16u * h);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] &= live;
        w[s] = __builtin_bit_cast(half8_t, v);
    }
}
__device__ __forceinline__ void moe_q8_block(half8_t (&w)[2], const uint8_t *row, uint32_t i, uint32_t h) {
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        uint32_t q0, q1;
        moe_get8(q0, q1, row + 8u * h, 34u * i + 2u + 16u * s);
        w[s] = mms_bytes<128>(q0 ^ 0x80808080u, q1 ^ 0x80808080u);
    }
}
// A byte holds elements j and j + 16, the pair of one conversion.
__device__ __forceinline__ void moe_mx_block(half8_t (&w)[2], const uint8_t *row, uint32_t i, uint32_t h, float scale, uint32_t live) {
    uint32_t q[2];
    moe_get8(q[0], q[1], row + 8u * h, 17u * i + 1u);
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        const uint32_t d = q[s] & live;
        moe_set(w[s], 0, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, scale, 0));
        moe_set(w[s], 2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, scale, 1));
        moe_set(w[s], 4, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, scale, 2));
        moe_set(w[s], 6, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, scale, 3));
    }
}
// (x & MASK) | over in one instruction, which takes no literal: the mask from a scalar register, which the
// compiler, left to know its value, puts back as a literal of an instruction of its own.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t moe_over(uint32_t x, uint32_t over) {
    uint32_t mask;
    asm("s_mov_b32 %0, %1" : "=s"(mask) : "i"(MASK));
    return (x & mask) | over;
}
__device__ __forceinline__ uint32_t moe_exponent() {  // under which a half's low bits are 1024 + the integer
    uint32_t v;
    asm("v_mov_b32 %0, 0x64006400" : "=v"(v));
    return v;
}
// Even blocks lie in the low nibbles, odd ones in the high nibbles of the same bytes. Under exponent 0x64 a low
// nibble q is 1024 + q and a high one in its place 1024 + 16 q: one fused multiply-add leaves q times the scale,
// exactly.
template <uint32_t TY>
__device__ __forceinline__ void moe_q45_block(half8_t (&w)[2], const uint8_t *row, uint32_t i, uint32_t h, uint32_t sc) {
    const bool high = i & 1u;
    const _Float16 f = (_Float16) (uint16_t) sc, m = high ? f * (_Float16) 0.0625f : f, a = f * (_Float16) (high ? -64.f : -1024.f);
    const uint32_t exponent = moe_exponent();
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        uint32_t q[2], hb[2] = {0u, 0u};
        moe_get8(q[0], q[1], row + 8u * h, (TY == 12 ? 16u : 48u) + 32u * (i >> 1) + 16u * s);
        if constexpr (TY == 13) moe_get8(hb[0], hb[1], row + 8u * h, 16u + 16u * s);
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (uint32_t odd = 0; odd < 2; ++odd) {  // bytes 0 and 2, 1 and 3
                const uint32_t x = odd ? q[d] >> 8 : q[d];
                uint32_t v = high ? moe_over<0x00F000F0u>(x, exponent) : moe_over<0x000F000Fu>(x, exponent);
                if constexpr (TY == 13) {  // the fifth bits: bit i of each byte, to bit 4 (8)
                    const uint32_t from = i + 8u * odd, to = high ? 8u : 4u;
                    const uint32_t y = from < to ? hb[d] << (to - from) : hb[d] >> (from - to);
                    v = high ? moe_over<0x01000100u>(y, v) : moe_over<0x00100010u>(y, v);
                }
                moe_set(w[s], 4 * d + 2 * (int) odd, __builtin_elementwise_fma(moe_h2(v), half2_t{m, m}, half2_t{a, a}));
            }
    }
}
// Q6_K, without the scales: q - 32
__device__ __forceinline__ void moe_q6_block(half8_t (&w)[2], const uint8_t *row, uint32_t i, uint32_t h) {
    const uint32_t exponent = moe_exponent();
#pragma unroll
    for (uint32_t s = 0; s < 2; ++s) {
        const uint32_t n = i >> 2, c = i & 3u, shl = 4u * (c >> 1), shh = 2u * c;
        uint32_t q[2], hb[2];
        moe_get8(q[0], q[1], row + 8u * h, 64u * n + 32u * (c & 1u) + 16u * s);
        moe_get8(hb[0], hb[1], row + 8u * h, 128u + 32u * n + 16u * s);
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (uint32_t odd = 0; odd < 2; ++odd) {
                const uint32_t from = shh + 8u * odd;
                const uint32_t y = from < 4u ? hb[d] << (4u - from) : hb[d] >> (from - 4u);
                const uint32_t v = moe_over<0x00300030u>(y, moe_over<0x000F000Fu>(q[d] >> (shl + 8u * odd), exponent));
                moe_set(w[s], 4 * d + 2 * (int) odd, moe_h2(v) - half2_t{(_Float16) 1056.f, (_Float16) 1056.f});
            }
    }
}

typedef __bf16 moe_bf8 __attribute__((ext_vector_type(8)));

// The reduction of one tile for a wave: acc[slot half][row tile], slots 32 and up only with BOTH. FOLD (MXFP4):
// the scales enter the operand; returns false where one is out of f16's range, and the sums are not valid then.
template <uint32_t TY, bool GU, int HALVES, int TS, int RT, bool BOTH, bool FOLD>
__device__ __forceinline__ bool moe_tile_sums(const MoeArgs &a, moe_f32x16 (&acc)[2][RT], uint8_t *xbuf, uint8_t *wbuf, uint16_t *sums,
                                              uint32_t e, const uint32_t *slots, uint32_t count, uint32_t r0) {
    using F = MoeTileFmt<TY, HALVES>;
    constexpr uint32_t WB = F::WB, SPW = WB / 2u;
    constexpr bool Q45 = TY == 12 || TY == 13, Q6 = TY == 14, MX = TY == 39, KQ = Q45 || Q6, PIPE = MX && TS == 2;
    constexpr int NT = BOTH ? 2 : 1;
    constexpr uint32_t WG = 2u * RT, DEPTH = TS == 1 ? 2u : 1u;  // weights are requested DEPTH windows ahead
    constexpr uint32_t XB = 2048u * TS, XPAIR = 2u * HALVES * XB;  // one half of a k-block, a pair of k-blocks
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 31u, h = lane >> 5;
    const uint32_t nb = a.cols / 32u, n_win = (nb + WB - 1u) / WB;
    // Window 0 has the first `head` blocks (it is copied whole, the rest of it belongs to window 1), the others WB each.
    const uint32_t head = nb - (n_win - 1u) * WB, steps0 = (head + 1u) / 2u, total = steps0 + (n_win - 1u) * SPW;
    auto wstart = [&](uint32_t w) __attribute__((always_inline)) { return w ? head + (w - 1u) * WB : 0u; };
    // Weights: copies of 16 rows each take four pieces per row, four lanes a row; what is left of a row's pieces is
    // copied for all rows at once (one piece), or 32 (two). The first half of the wave's rows are of matrix 0 from r0, the
    // second of matrix 1 from r0 (GU) or matrix 0 from r0 + 16 RT; rows past the last repeat it. A lane's offset
    // within the matrix is 32 bits (64 rows of at most 2 MiB), the rest of the address is the wave's.
    constexpr uint32_t NQ = F::NP % 4u == 3u ? F::NP / 4u + 1u : F::NP / 4u, LEFT = F::NP % 4u == 3u ? 0u : F::NP % 4u;
    constexpr uint32_t NR = LEFT == 2u ? RT : LEFT;  // copies of what is left
    constexpr uint32_t RB = F::S % 16u == 8u ? 8u : 16u;  // bytes of the last piece that are new
    static_assert(RB == 16u || LEFT == 1u, "a short last piece stands alone");
    const uint32_t wr0 = min(r0, a.rows - 1u), wleft = a.rows - 1u - wr0;
    const uint8_t *const wrow0 = a.w[0] + e * a.expert_bytes + (uint64_t) wr0 * a.row_bytes;
    const uint8_t *const wrow1 = GU ? a.w[1] + e * a.expert_bytes + (uint64_t) wr0 * a.row_bytes : wrow0;
    const uint32_t rbytes = (uint32_t) a.row_bytes;
    uint32_t woff[WG], roff[NR ? NR : 1];
#pragma unroll
    for (uint32_t g = 0; g < WG; ++g) woff[g] = min((lane >> 2) + 16u * (GU ? g % RT : g), wleft) * rbytes;
    // row of the wave that a lane copies what is left of
    auto rrow = [&](uint32_t g) __attribute__((always_inline)) { return LEFT == 1u ? lane % (32u * RT) : (lane >> 1) + 32u * g; };
#pragma unroll
    for (uint32_t g = 0; g < NR; ++g)
        roff[g] = min(GU ? rrow(g) % (16u * RT) : rrow(g), wleft) * rbytes + min(64u * NQ + 16u * (LEFT == 1u ? 0u : lane & 1u), F::S - RB);
    u32x4_t wreg[DEPTH][WG][NQ], rreg[DEPTH][NR ? NR : 1];
    auto wload = [&](uint32_t w, uint32_t set) __attribute__((always_inline)) {
        const uint64_t o = (uint64_t) wstart(w) * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
#pragma unroll
        for (uint32_t g = 0; g < WG; ++g)
#pragma unroll
            for (uint32_t k = 0; k < NQ; ++k) {
                // only the last quad can pass the window's end, by pieces that repeat the one before
                const uint32_t at = 64u * (k + 1u) <= F::S ? 64u * k + 16u * (lane & 3u) : min(64u * k + 16u * (lane & 3u), F::S - 16u);
                __builtin_memcpy(&wreg[set][g][k], (g < RT ? wrow0 : wrow1) + o + (woff[g] + at), 16);
            }
#pragma unroll
        for (uint32_t g = 0; g < NR; ++g)
            __builtin_memcpy(&rreg[set][g], (rrow(g) < 16u * RT ? wrow0 : wrow1) + o + roff[g], RB);
    };
    auto put16 = [&](uint8_t *d, u32x4_t v) __attribute__((always_inline)) {
        if constexpr (TY == 1) {
            *(u32x4_t *) d = v;
        } else {
            *(u32x2_t *) d = u32x2_t{v[0], v[1]};
            *(u32x2_t *) (d + 8) = u32x2_t{v[2], v[3]};
        }
    };
    auto wput = [&](uint32_t set) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t g = 0; g < WG; ++g)
#pragma unroll
            for (uint32_t k = 0; k < NQ; ++k) {
                const uint32_t piece = 4u * k + (lane & 3u);
                put16(wbuf + ((lane >> 2) + 16u * g) * F::RS + 16u * (4u * (k + 1u) <= F::NP ? piece : min(piece, F::NP - 1u)), wreg[set][g][k]);
            }
#pragma unroll
        for (uint32_t g = 0; g < NR; ++g) {
            uint8_t *d = wbuf + rrow(g) * F::RS + 64u * NQ + 16u * (LEFT == 1u ? 0u : lane & 1u);
            if constexpr (RB == 8u) *(u32x2_t *) d = u32x2_t{rreg[set][g][0], rreg[set][g][1]};
            else put16(d, rreg[set][g]);
        }
    };
    // inputs: thread i, load (half, group g): slot i / 8 + 32 g, 16 bytes i % 8 of the pair's 128
    const uint16_t *xrow[NT];
#pragma unroll
    for (uint32_t g = 0; g < NT; ++g)
        xrow[g] = (const uint16_t *) a.x + (uint64_t) (slots[min((tid >> 3) + 32u * g, count - 1u)] / a.x_div) * a.cols + 8u * (tid & 7u);
    const int64_t xlo = HALVES == 2 ? (const uint16_t *) a.x_lo - (const uint16_t *) a.x : 0;
    u32x4_t xreg[HALVES][NT];
    auto xload = [&](uint32_t step) __attribute__((always_inline)) {
        const uint32_t b = min(step < steps0 ? 2u * step : head + 2u * (step - steps0), nb - 2u);
#pragma unroll
        for (uint32_t g = 0; g < NT; ++g)
#pragma unroll
            for (int f = 0; f < HALVES; ++f) __builtin_memcpy(&xreg[f][g], xrow[g] + (f ? xlo : 0) + 32u * b, 16);
    };
    auto xput = [&](uint32_t buf) __attribute__((always_inline)) {
        const uint32_t blk = (tid >> 2) & 1u, c = tid & 3u;
#pragma unroll
        for (uint32_t g = 0; g < NT; ++g) {
            const uint32_t u = (tid >> 3) + 32u * g;
#pragma unroll
            for (int f = 0; f < HALVES; ++f)
                *(u32x4_t *) (xbuf + buf * XPAIR + (blk * HALVES + f) * XB + u * 64u + 16u * (c ^ moe_swz(u))) = xreg[f][g];
        }
    };
    // The sums of x over the k-blocks of the pair in the registers, as this thread's bf16 piece: piece
    // tid % 4 of block (tid / 4) % 2, slots tid / 8 and + 32. Cut off bits, so that three pieces are exact.
    auto xsums = [&](uint32_t (&piece)[NT]) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t g = 0; g < NT; ++g) {
            float s = 0.f, one = 1.f;
            asm("" : "+v"(one));  // s + v as a mixed-precision multiply-add, without a conversion
#pragma unroll
            for (int f = HALVES - 1; f >= 0; --f) {
                const half8_t v = __builtin_bit_cast(half8_t, xreg[f][g]);
#pragma unroll
                for (int k = 0; k < 8; ++k) s = fmaf((float) v[k], one, s);
            }
            s += dpp<0xB1>(s);
            s += dpp<0x4E>(s);
            const uint32_t p0 = __float_as_uint(s) & 0xFFFF0000u;
            const float s1 = s - __uint_as_float(p0);
            const uint32_t p1 = __float_as_uint(s1) & 0xFFFF0000u;
            const uint32_t p2 = __float_as_uint(s1 - __uint_as_float(p1));
            const uint32_t c = tid & 3u;
            piece[g] = (c == 0u ? p0 : c == 1u ? p1 : c == 2u ? p2 : 0u) >> 16;
        }
    };
    auto sput = [&](const uint32_t (&piece)[NT], uint32_t pair) __attribute__((always_inline)) {  // `pair` of the window
#pragma unroll
        for (uint32_t g = 0; g < NT; ++g)
            sums[((tid >> 3) + 32u * g) * 32u + (tid & 3u) * 8u + 2u * pair + ((tid >> 2) & 1u)] = (uint16_t) piece[g];
    };

#pragma unroll
    for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[tt][rt][j] = 0.f;
    // K-quants: per row tile, what the accumulators are in units of, the factor of the super-block in LDS, and
    // whether that counts at all (0: its scales are taken as 0, and the unit stays)
    float unit[2] = {1.f, 1.f}, factor[2] = {1.f, 1.f};
    bool ok = true;

    auto mul = [&](const half8_t &x, const half8_t &w, const moe_f32x16 &c) __attribute__((always_inline)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w, c, 0, 0, 0);
    };
    // One k-block's weights for the matrix cores: [row tile][slice], scales that stayed out, and what Q6_K's
    // rounding lost
    struct Ops {
        half8_t w[RT][2], lost[Q6 ? RT : 1][2];
        float f[2];
        bool any[2];
    };
    auto decode = [&](Ops &o, uint32_t i, uint32_t live) __attribute__((always_inline)) {  // k-block i of the window
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint8_t *row = wbuf + (32u * rt + n) * F::RS;
            if constexpr (TY == 1) {
                moe_f16_block(o.w[rt], row, i, h, live);
            } else if constexpr (TY == 8) {
                moe_q8_block(o.w[rt], row, i, h);
                o.f[rt] = live ? mms_f16(*(const uint16_t *) (row + 34u * i)) : 0.f;
            } else if constexpr (MX) {
                const uint32_t e8 = row[17u * i];
                o.f[rt] = __uint_as_float(FOLD || e8 ? e8 << 23 : 0x00400000u);  // 2^(e - 127)
                moe_mx_block(o.w[rt], row, i, h, FOLD ? o.f[rt] : 1.f, live);
            } else if constexpr (Q45) {
                const u32x2_t h0 = *(const u32x2_t *) row, h1 = *(const u32x2_t *) (row + 8);
                moe_q45_block<TY>(o.w[rt], row, i, h, factor[rt] != 0.f ? moe_k4_scale(u32x4_t{h0[0], h0[1], h1[0], h1[1]}, i) : 0u);
            } else {
                moe_q6_block(o.w[rt], row, i, h);
                const uint32_t sc = *(const uint16_t *) (row + 192u + 2u * i);
                uint32_t bits = 0u;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const _Float16 m = factor[rt] != 0.f ? (_Float16) (int16_t) (int8_t) (sc >> (8 * s)) : (_Float16) 0.f;
                    const half8_t q = o.w[rt][s];
                    o.w[rt][s] = moe_times(q, m);
                    o.lost[rt][s] = moe_lost(q, m, o.w[rt][s]);
                    const u32x4_t v = __builtin_bit_cast(u32x4_t, o.lost[rt][s]);
                    bits |= (v[0] | v[1] | v[2] | v[3]) & 0x7FFF7FFFu;
                }
                o.any[rt] = __ballot(bits != 0u) != 0ull;  // some product of the wave was rounded
            }
        }
    };
    auto products = [&](uint32_t buf, uint32_t blk, const Ops &o) __attribute__((always_inline)) {  // block blk of the pair in buffer buf
        half8_t x[HALVES][NT][2];
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int g = 0; g < HALVES; ++g) {
                    const uint32_t u = 32u * tt + n;
                    x[g][tt][s] = __builtin_bit_cast(half8_t, *(const u32x4_t *) (xbuf + buf * XPAIR + (blk * HALVES + g) * XB +
                                                                                  u * 64u + 16u * ((2u * s + h) ^ moe_swz(u))));
                }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (TY == 1 || KQ || FOLD) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int g = 0; g < HALVES; ++g)
#pragma unroll
                        for (int tt = 0; tt < NT; ++tt) acc[tt][rt] = mul(x[g][tt][s], o.w[rt][s], acc[tt][rt]);
                if constexpr (Q6)
                    if (o.any[rt]) {
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int tt = 0; tt < NT; ++tt) acc[tt][rt] = mul(x[0][tt][s], o.lost[rt][s], acc[tt][rt]);
                    }
            } else {
                moe_f32x16 d[NT];
#pragma unroll
                for (int tt = 0; tt < NT; ++tt) d[tt] = moe_f32x16{};
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int g = 0; g < HALVES; ++g)
#pragma unroll
                        for (int tt = 0; tt < NT; ++tt) d[tt] = mul(x[g][tt][s], o.w[rt][s], d[tt]);
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[tt][rt][j] = fmaf(o.f[rt], d[tt][j], acc[tt][rt][j]);
            }
        }
    };
    // the next window into LDS, when the last one's weights have all been taken from there, and the one after it
    // requested
    auto advance = [&](uint32_t w, uint32_t set) __attribute__((always_inline)) {  // set: w % DEPTH
        __builtin_amdgcn_wave_barrier();
        wput(set);
        __builtin_amdgcn_wave_barrier();
        wload(min(w + DEPTH, n_win - 1u), set);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (KQ) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                factor[rt] = mms_f16(*(const uint16_t *) (wbuf + (32u * rt + n) * F::RS + (Q6 ? 208u + MmsFmt<14>::LAST : 0u)));
        }
        if constexpr (FOLD) {
            uint32_t lo = 255u, hi = 0u;  // of one row per lane
#pragma unroll
            for (uint32_t i = 0; i < WB; ++i) {
                const uint32_t e8 = wbuf[lane % (32u * RT) * F::RS + 17u * i];
                lo = min(lo, e8);
                hi = max(hi, e8);
            }
            ok = ok && lo >= 114u && hi <= 139u;
        }
    };
    // the accumulators from the last super-block's unit to this one's
    auto rescale = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float ratio = factor[rt] != 0.f ? unit[rt] / factor[rt] : 1.f;
            unit[rt] = factor[rt] != 0.f ? factor[rt] : unit[rt];
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[tt][rt][j] *= ratio;
        }
    };
    auto mins = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint8_t *row = wbuf + (32u * rt + n) * F::RS;
            const u32x2_t h0 = *(const u32x2_t *) row, h1 = *(const u32x2_t *) (row + 8);
            const u32x4_t hd = {h0[0], h0[1], h1[0], h1[1]};
            const float f = -mms_f16(hd[0] >> 16) / unit[rt];
            moe_bf8 m;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) m[k] = (__bf16) (float) moe_k4_min(hd, k);
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                moe_f32x16 d = {};
#pragma unroll
                for (uint32_t p = 0; p < 2; ++p)
                    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        __builtin_bit_cast(moe_bf8, *(const u32x4_t *) (sums + (32u * tt + n) * 32u + 16u * p + 8u * h)), m, d, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[tt][rt][j] = fmaf(f, d[j], acc[tt][rt][j]);
            }
        }
    };

    uint32_t piece[NT] = {}, step = 0;
    // the step's copies: the next pair of inputs into the other buffer (after the last: nothing reads it), the one
    // after it requested
    auto copies = [&]() __attribute__((always_inline)) {
        xput((step + 1u) & 1u);
        if constexpr (Q45) xsums(piece);
        xload(min(step + 2u, total - 1u));
        __builtin_amdgcn_sched_barrier(0);  // left alone, the loads sink to the step's end, and the next waits for them
    };
    const uint32_t all = 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t d = 0; d < DEPTH; ++d) wload(min(d, n_win - 1u), d);
    xload(0u);
    xput(0u);
    if constexpr (Q45) xsums(piece);
    xload(min(1u, total - 1u));
    moe_barrier();
    advance(0u, 0u);
    Ops A, B;
    uint32_t w = 0;
    // Sums: the pair that is stored for the next step has its own stored with it, but the next window's first pair
    // waits for that window, when the mins of this one have been taken.
    auto window = [&](uint32_t w, uint32_t next_set) __attribute__((always_inline)) {
        const uint32_t blocks = w ? WB : head;
        if constexpr (KQ) rescale();
#pragma unroll
        for (uint32_t j = 0; j < SPW; ++j) {
            if (!KQ && 2u * j >= blocks) continue;
            const uint32_t live = KQ || 2u * j + 1u < blocks ? all : 0u;
            if constexpr (Q45)
                if (j == 0) sput(piece, 0u);
            copies();
            if constexpr (Q45)
                if (j + 1u < SPW) sput(piece, j + 1u);
            decode(A, 2u * j, all);
            decode(B, 2u * j + 1u, live);
            products(step & 1u, 0u, A);
            products(step & 1u, 1u, B);
            if constexpr (Q45)
                if (j + 1u == SPW) mins();
            moe_barrier();
            ++step;
        }
        advance(w + 1u, next_set);
    };
    if (!PIPE || head < WB) {
        const uint32_t until = PIPE ? 1u : n_win;
#pragma unroll 1
        for (; w < until; w += DEPTH) {
            window(w, 1u % DEPTH);
            if constexpr (DEPTH == 2u)
                if (w + 1u < until) window(w + 1u, 0u);
        }
    }
    // MXFP4's whole windows: each block's weights are decoded while the one before is multiplied (the other formats
    // have no registers left for it: Q4_K 153 -> 167 us, Q8_0 130 -> 154)
    if constexpr (PIPE) {
        decode(A, 0u, all);
#pragma unroll 1
        for (; w < n_win; ++w) {
#pragma unroll
            for (uint32_t j = 0; j < SPW; ++j) {
                copies();
                decode(B, 2u * j + 1u, all);
                products(step & 1u, 0u, A);
                if (j + 1u == SPW) advance(w + 1u, 0u);
                decode(A, (2u * j + 2u) % WB, all);
                products(step & 1u, 1u, B);
                moe_barrier();
                ++step;
            }
        }
    }
    if constexpr (KQ) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[tt][rt][j] *= unit[rt];
    }
    return ok;
}

template <uint32_t TY, bool GU, int HALVES, int TS, int RT, bool BOTH>
__device__ __forceinline__ void moe_tile_half(const MoeArgs &a, uint8_t *xbuf, uint8_t *wbuf, uint16_t *sums, uint32_t e,
                                              const uint32_t *slots, uint32_t count, uint32_t r0) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 31u, h = lane >> 5;
    moe_f32x16 acc[2][RT];
    const bool ok = moe_tile_sums<TY, GU, HALVES, TS, RT, BOTH, TY == 39>(a, acc, xbuf, wbuf, sums, e, slots, count, r0);
    if constexpr (TY == 39)  // some scale out of range: again, every block's sum scaled by itself
        if (__syncthreads_or(!ok))
            (void) moe_tile_sums<TY, GU, HALVES, TS, RT, BOTH, false>(a, acc, xbuf, wbuf, sums, e, slots, count, r0);
    // Each lane holds one slot of the tile, from where the others take it (read from memory beside each store, they
    // were a round trip apiece: a product of 200 tiles of 1536 x 512 Q4_K 69 us, now 61).
    const uint32_t held = slots[min(lane, count - 1u)];
#pragma unroll
    for (int rt = 0; rt < (GU ? 1 : RT); ++rt) {
        // GU: gate and up in the lane's two row tiles, or, of one tile, in lanes 16 apart, the first 16 of which go on
        const uint32_t r = r0 + (GU && RT == 1 ? n & 15u : 32u * rt + n);
        const bool in = r < a.rows && (!GU || RT == 2 || n < 16u);
        const uint64_t at_row = (uint64_t) e * a.rows + min(r, a.rows - 1u);
        const float b0 = a.bias[0] ? a.bias[0][at_row] : 0.f, b1 = GU && a.bias[1] ? a.bias[1][at_row] : 0.f;
        // GU: where the next product, whose weights are of type a.y_order, looks for column r (it has whole blocks)
        const uint32_t col = GU ? (r & ~31u) | moe_place(a.y_order, r & 31u) : r;
#pragma unroll
        for (int tt = 0; tt < (BOTH ? 2 : 1); ++tt)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t u = 32u * tt + 8u * (j >> 2) + 4u * h + (j & 3);
                const uint64_t o = (uint64_t) (uint32_t) __shfl((int) held, (int) u) * a.rows + col;
                const float up = !GU ? 0.f : RT == 2 ? acc[tt][RT - 1][j] : __shfl_xor(acc[tt][0][j], 16);
                if (!in || u >= count) continue;
                if constexpr (GU) {
                    const float v = moe_activation(a, acc[tt][0][j] + b0, up + b1);
                    const _Float16 hi = (_Float16) v;
                    ((_Float16 *) a.y)[o] = hi;
                    if constexpr (HALVES == 2) ((_Float16 *) a.y_lo)[o] = (_Float16) (v - (float) hi);
                } else {
                    const float v = acc[tt][rt][j] + b0;
                    if (a.y_f16) ((_Float16 *) a.y)[o] = (_Float16) v;
                    else ((float *) a.y)[o] = v;
                }
            }
    }
}

// Tiles of up to 32 TS slots, RT row tiles of 32 per wave.
template <uint32_t TY, bool GU, int HALVES, int TS, int RT>
__device__ __forceinline__ void moe_tile_body(const MoeArgs &a) {
    using F = MoeTileFmt<TY, HALVES>;
    __shared__ __attribute__((aligned(1024))) uint8_t xbuf[4 * HALVES * 2048 * TS];
    __shared__ __attribute__((aligned(16))) uint8_t wbuf[4][32 * RT * F::RS];
    // Q4_K, Q5_K: [slot][piece 0 .. 3][block of the super-block] bf16, a block's sum of x in three pieces
    __shared__ __attribute__((aligned(16))) uint16_t sums[TY == 12 || TY == 13 ? 32 * TS * 32 : 8];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The work in the order (expert, row tile, tile of slots), cut into eight equal runs, one for each XCD
    // (work-group i is on XCD i % 8): an expert's rows are then read by the L2 that all of its tiles go through, and
    // a tile's inputs by one or two of them.
    const uint32_t items = *a.n_tiles * a.row_tiles, run = (items + 7u) / 8u;
    const uint32_t at = (blockIdx.x & 7u) * run + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= run || at >= items) return;
    const MoeTile some = a.tiles[at / a.row_tiles];  // a tile of the expert
    const uint32_t tile0 = at / a.row_tiles - some.index, in = at - tile0 * a.row_tiles;
    const uint32_t rt_i = __builtin_amdgcn_readfirstlane(in / some.of);
    const MoeTile t = a.tiles[tile0 + in % some.of];
    const uint32_t e = __builtin_amdgcn_readfirstlane(t.expert), count = __builtin_amdgcn_readfirstlane(t.count);
    const uint32_t *const slots = a.list + t.first;
    // this wave's rows: 32 RT from r0, GU: half as many of each matrix
    constexpr uint32_t ROWS = 32u * RT / (GU ? 2u : 1u);
    const uint32_t r0 = (4u * rt_i + wave) * ROWS;
    if (e == a.n_expert) {
        if (!GU && a.zero_skipped)
            for (uint32_t u = 0; u < count; ++u) {
                const uint64_t o = (uint64_t) slots[u] * a.rows + r0 + lane;
                if (lane >= ROWS || r0 + lane >= a.rows) continue;
                if (a.y_f16) ((uint16_t *) a.y)[o] = 0;
                else ((float *) a.y)[o] = 0.f;
            }
        return;
    }
    if constexpr (TS == 2)
        if (count > 32u) return moe_tile_half<TY, GU, HALVES, TS, RT, true>(a, xbuf, wbuf[wave], sums, e, slots, count, r0);
    moe_tile_half<TY, GU, HALVES, TS, RT, false>(a, xbuf, wbuf[wave], sums, e, slots, count, r0);
}

}  // namespace

// Shapes, as moe_tile_rows (runtime_moe.h) has them. Wide tiles, 64 slots x 64 rows a wave and two waves per SIMD, decode
// each weight for twice the slots and read the inputs half as often; narrow ones, 32 rows a wave, hold three or four
// waves per SIMD, which cover each other's waits. Products measured wide, narrow (us):
//   MXFP4 f32 361 / 369, f16 172 / 162; Q4_K f32 174 / 201, f16 170 / 169; Q5_K 202 / 225; Q6_K f32 390 / 304,
//   f16 162 / 134; Q8_0 200 / 189; F16 f32 165 / 161, f16 286 / 260
// Light tiles, of 32 slots, for few slots an expert: four waves where the registers allow it without spilling
// (MXFP4: 24 tokens of 128 experts 133 + 82 us, with three 135 + 86; Q8_0, 200 tokens of 64 experts: 130 + 78, with
// three 114 + 62).
#define MOE_TILE_KERNEL(NAME, TY, KIND, GU, IO, HALVES, RT, WAVES, LIGHT_WAVES)                                     \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))            \
    moearc_moe_tile_##NAME##_##KIND##_##IO##_k(MoeArgs a) { moe_tile_body<TY, GU, HALVES, 2, RT>(a); }              \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(LIGHT_WAVES, LIGHT_WAVES))) \
    moearc_moe_light_##NAME##_##KIND##_##IO##_k(MoeArgs a) { moe_tile_body<TY, GU, HALVES, 1, 1>(a); }
#define MOE_TILE(NAME, TY, RT32, WAVES32, RT16, WAVES16, LIGHT_WAVES)          \
    MOE_TILE_KERNEL(NAME, TY, gu, true, f32, 2, RT32, WAVES32, LIGHT_WAVES)    \
    MOE_TILE_KERNEL(NAME, TY, gu, true, f16, 1, RT16, WAVES16, LIGHT_WAVES)    \
    MOE_TILE_KERNEL(NAME, TY, p, false, f32, 2, RT32, WAVES32, LIGHT_WAVES)    \
    MOE_TILE_KERNEL(NAME, TY, p, false, f16, 1, RT16, WAVES16, LIGHT_WAVES)
MOE_TILE(f16, 1, 1, 4, 1, 4, 4)
MOE_TILE(q8_0, 8, 1, 3, 1, 3, 3)
MOE_TILE(q4_k, 12, 2, 2, 2, 2, 3)
MOE_TILE(q5_k, 13, 2, 2, 2, 2, 3)
MOE_TILE(q6_k, 14, 1, 3, 1, 3, 3)
MOE_TILE(mxfp4, 39, 2, 2, 1, 3, 4)
