// The experts' products over a plan (MoeArgs): tiles of up to 64 of one expert's slots times 256 weight rows
// (128 of gate and the same 128 of up), on v_mfma_f32_32x32x16_f16.
//
// The product is computed transposed, D[slot][row], so that a lane holds one weight row in all of its
// accumulators and a block's scale is one per-lane factor. Work-group: 4 waves, each the tile's 64 slots
// times 64 rows of its own as 2 x 2 tiles of 32 x 32 (gate_up: rows of gate beside the same rows of up, so
// the activation needs no exchange). A weight is thus decoded by one wave only, and the slots' inputs, four
// bytes an element where the weights have half to one, are shared by 256 rows. Tiles of at most 32 slots
// skip the second half.
// - Weights: windows of WB k-blocks move through registers (the next window in flight while this one is
//   multiplied) into the wave's LDS; lane l copies 16-byte pieces of rows 32 (l / 32) .. + 31.
// - Inputs: pairs of k-blocks, f16 (hi and lo), 64 bytes per slot and block, whose 16-byte chunk c (k 8c ..)
//   is at c ^ swz(slot); two buffers, the pair after the next in registers; one barrier per pair.
//
// Scales cost a vector instruction per accumulator and k-block beside 32 cycles of MFMA, so where the
// formats allow they are part of the operand, exactly, and the accumulators run through:
// - MXFP4: 2^(e - 127) scales the E2M1 code in the conversion, exact while every product is a normal f16,
//   which is checked per window (e from 114 to 139); other windows scale each block's f32 sum.
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

template <uint32_t TY>
struct MoeTileFmt {
    static constexpr uint32_t WB = TY == 1 ? 2 : TY == 8 ? 4 : 8;
    static constexpr uint32_t S = WB * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
    static constexpr uint32_t NP = (S + 15u) / 16u;       // 16-byte pieces of a row's window
    static constexpr uint32_t RS = 16u * (NP | 1u);       // an odd number of them apart: rows on all banks
    static constexpr bool SPLIT_LAST = TY == 8;           // as MoeFmt
};

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

// Eight elements of k-block i of a row's window in LDS, k 8 lq .. 8 lq + 7: the payload as f16 integers
// (E2M1 values times `scale` for MXFP4).
template <uint32_t TY>
__device__ __forceinline__ half8_t moe_payload(const uint8_t *row, uint32_t i, uint32_t lq, float scale) {
    uint32_t q0, q1;
    if constexpr (TY == 39) {
        mms_get8(q0, q1, row, 17u * i + 1u + (i == 7u ? MmsFmt<39>::LAST : 0u), lq & 1u);
        const uint32_t q[2] = {q0, q1};
        half8_t r;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t x = (q[j] >> (4u * (lq >> 1))) & 0x0F0F0F0Fu;
            const uint32_t y = x | (x >> 4);  // pairs in bytes 0 and 2
            const half2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(y, scale, 0);
            const half2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(y, scale, 2);
            r[4 * j] = p0[0];
            r[4 * j + 1] = p0[1];
            r[4 * j + 2] = p1[0];
            r[4 * j + 3] = p1[1];
        }
        return r;
    } else if constexpr (TY == 12 || TY == 13) {
        mms_get8(q0, q1, row, (TY == 12 ? 16u : 48u) + 32u * (i >> 1), lq);
        const uint32_t sh = 4u * (i & 1u);
        q0 = (q0 >> sh) & 0x0F0F0F0Fu;
        q1 = (q1 >> sh) & 0x0F0F0F0Fu;
        if constexpr (TY == 13) {
            uint32_t h0, h1;
            mms_get8(h0, h1, row, 16u, lq);
            q0 |= ((h0 >> i) & 0x01010101u) << 4;
            q1 |= ((h1 >> i) & 0x01010101u) << 4;
        }
        return mms_bytes<0>(q0, q1);
    } else {
        static_assert(TY == 14, "a format whose scale enters the operand");
        const uint32_t n = i >> 2, c = i & 3u, shl = 4u * (c >> 1), shh = 2u * c;
        uint32_t h0, h1;
        mms_get8(q0, q1, row, 64u * n + 32u * (c & 1u), lq);
        mms_get8(h0, h1, row, 128u + 32u * n, lq);
        return mms_bytes<32>(((q0 >> shl) & 0x0F0F0F0Fu) | (((h0 >> shh) & 0x03030303u) << 4),
                             ((q1 >> shl) & 0x0F0F0F0Fu) | (((h1 >> shh) & 0x03030303u) << 4));
    }
}

typedef __bf16 moe_bf8 __attribute__((ext_vector_type(8)));

template <uint32_t TY, bool GU, int HALVES>
__device__ __forceinline__ void moe_tile_body(const MoeArgs &a) {
    using F = MoeTileFmt<TY>;
    constexpr uint32_t WB = F::WB, SPW = WB / 2u;
    constexpr bool Q45 = TY == 12 || TY == 13, Q6 = TY == 14, MX = TY == 39;
    constexpr bool KQ = Q45 || Q6;
    constexpr uint32_t XB = 4096u, XPAIR = 2u * HALVES * XB;  // one half of a k-block, a pair of k-blocks
    __shared__ __attribute__((aligned(1024))) uint8_t xbuf[2 * XPAIR];
    __shared__ __attribute__((aligned(16))) uint8_t wbuf[4][64 * F::RS];
    // Q4_K, Q5_K: [slot][piece 0 .. 3][block of the super-block] bf16, a block's sum of x in three pieces
    __shared__ __attribute__((aligned(16))) uint16_t sums[Q45 ? 64 * 32 : 8];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31u, h = lane >> 5;

    const uint32_t ti = blockIdx.x / a.row_tiles, rt_i = blockIdx.x % a.row_tiles;
    if (ti >= *a.n_tiles) return;
    const MoeTile t = a.tiles[ti];
    const uint32_t e = __builtin_amdgcn_readfirstlane(t.expert), count = __builtin_amdgcn_readfirstlane(t.count);
    const uint32_t *const slots = a.list + t.first;
    // this wave's rows: GU: 32 of each matrix from r0, else 64 from r0
    const uint32_t r0 = rt_i * (GU ? 128u : 256u) + wave * (GU ? 32u : 64u);
    if (e == a.n_expert) {
        if (!GU && a.zero_skipped)
            for (uint32_t u = 0; u < count; ++u) {
                const uint64_t o = (uint64_t) slots[u] * a.rows + r0 + lane;
                if (r0 + lane >= a.rows) continue;
                if (a.y_f16) ((uint16_t *) a.y)[o] = 0;
                else ((float *) a.y)[o] = 0.f;
            }
        return;
    }
    const bool both = count > 32u;  // uniform
    const uint32_t nb = a.cols / 32u, n_win = (nb + WB - 1u) / WB, total = n_win * SPW;
    // window w starts at block min(w WB, nb - WB): the last one may repeat blocks, which are skipped
    auto wstart = [&](uint32_t w) { return min(w * WB, nb - WB); };

    // weights: lane l's pieces l % 32 + 32 j of rows r0 + 32 (l / 32) .. (GU: of matrix l / 32)
    const uint8_t *wsrc = a.w[GU ? h : 0] + e * a.expert_bytes;
    const uint32_t wr0 = min(r0 + (GU ? 0u : 32u * h), a.rows - 1u), wleft = a.rows - 1u - wr0;
    wsrc += (uint64_t) wr0 * a.row_bytes;
    u32x4_t wreg[F::NP];
    auto wload = [&](uint32_t w) {
        const uint8_t *p = wsrc + (uint64_t) wstart(w) * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
#pragma unroll
        for (uint32_t j = 0; j < F::NP; ++j) {
            const uint32_t q = n + 32u * j, row = q / F::NP, piece = q % F::NP;
            __builtin_memcpy(&wreg[j], p + (uint64_t) min(row, wleft) * a.row_bytes + min(16u * piece, F::S - 16u), 16);
        }
    };
    auto wput = [&]() {
#pragma unroll
        for (uint32_t j = 0; j < F::NP; ++j) {
            const uint32_t q = n + 32u * j, row = q / F::NP, piece = q % F::NP;
            uint8_t *d = wbuf[wave] + (32u * h + row) * F::RS;
            if constexpr (F::SPLIT_LAST) {
                d += min(16u * piece, F::S - 16u);
                *(u32x2_t *) d = u32x2_t{wreg[j][0], wreg[j][1]};
                *(u32x2_t *) (d + 8) = u32x2_t{wreg[j][2], wreg[j][3]};
            } else {
                *(u32x4_t *) (d + 16u * piece) = wreg[j];
            }
        }
    };
    // inputs: thread i, load (half, group g): slot i / 8 + 32 g, 16 bytes i % 8 of the pair's 128
    const uint16_t *xrow[2];
#pragma unroll
    for (uint32_t g = 0; g < 2; ++g)
        xrow[g] = (const uint16_t *) a.x + (uint64_t) (slots[min((tid >> 3) + 32u * g, count - 1u)] / a.x_div) * a.cols + 8u * (tid & 7u);
    const int64_t xlo = HALVES == 2 ? (const uint16_t *) a.x_lo - (const uint16_t *) a.x : 0;
    u32x4_t xreg[HALVES][2];
    auto xload = [&](uint32_t step) {
        const uint32_t b = wstart(step / SPW) + 2u * (step % SPW);
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
            if (g == 0u || both)
#pragma unroll
                for (int f = 0; f < HALVES; ++f)
                    __builtin_memcpy(&xreg[f][g], xrow[g] + (f ? xlo : 0) + 32u * b, 16);
    };
    auto xput = [&](uint32_t buf) {
        const uint32_t blk = (tid >> 2) & 1u, c = tid & 3u;
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
            if (g == 0u || both) {
                const uint32_t u = (tid >> 3) + 32u * g;
#pragma unroll
                for (int f = 0; f < HALVES; ++f)
                    *(u32x4_t *) (xbuf + buf * XPAIR + (blk * HALVES + f) * XB + u * 64u + 16u * (c ^ moe_swz(u))) = xreg[f][g];
            }
    };
    // The sums of x over the k-blocks of the pair in the registers, as this thread's bf16 piece: piece
    // tid % 4 of block (tid / 4) % 2, slots tid / 8 and + 32. Cut off bits, so that three pieces are exact.
    auto xsums = [&](uint32_t (&piece)[2]) {
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
            if (g == 0u || both) {
                float s = 0.f;
#pragma unroll
                for (int f = HALVES - 1; f >= 0; --f) {
                    const half8_t v = __builtin_bit_cast(half8_t, xreg[f][g]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) s += (float) v[k];
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
    auto sput = [&](const uint32_t (&piece)[2], uint32_t pair) {  // `pair` of the window
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
            if (g == 0u || both)
                sums[((tid >> 3) + 32u * g) * 32u + (tid & 3u) * 8u + 2u * pair + ((tid >> 2) & 1u)] = (uint16_t) piece[g];
    };

    moe_f32x16 acc[2][2];  // [slot half][row tile]
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[tt][rt][j] = 0.f;

    // K-quants: per row tile, what the accumulators are in units of, and whether the super-block counts at
    // all (d = 0: its scales are taken as 0, and the unit stays)
    float unit[2] = {1.f, 1.f};
    bool counts[2] = {true, true};

    bool fold = false;  // MXFP4: this window's scales are in the operand
    auto mul = [&](const half8_t &x, const half8_t &w, const moe_f32x16 &c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w, c, 0, 0, 0);
    };
    // k-block i of the window, block blk of the pair in buffer buf
    auto compute = [&](uint32_t buf, uint32_t blk, uint32_t i) {
        half8_t x[HALVES][2][2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
            if (tt == 0 || both)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int f = 0; f < HALVES; ++f) {
                        const uint32_t u = 32u * tt + n;
                        x[f][tt][s] = __builtin_bit_cast(half8_t, *(const u32x4_t *) (xbuf + buf * XPAIR + (blk * HALVES + f) * XB +
                                                                                      u * 64u + 16u * ((2u * s + h) ^ moe_swz(u))));
                    }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const uint8_t *row = wbuf[wave] + (32u * rt + n) * F::RS;
            half8_t w[2], wl[2];
            float s0 = 0.f, s1 = 0.f;
            bool lost = false;  // Q6_K: some product of the wave was rounded
            if constexpr (Q45) {
                const uint32_t sc = counts[rt] ? moe_k4_scale(*(const u32x4_t *) row, i) : 0u;
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    w[s] = moe_times(moe_payload<TY>(row, i, 2u * s + h, 1.f), (_Float16) (uint16_t) sc);
            } else if constexpr (Q6) {
                const uint32_t sc = *(const uint16_t *) (row + 192u + 8u * (i >> 2) + 2u * (i & 3u));
                uint32_t any = 0u;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const _Float16 f = counts[rt] ? (_Float16) (int16_t) (int8_t) (sc >> (8 * s)) : (_Float16) 0.f;
                    const half8_t q = moe_payload<TY>(row, i, 2u * s + h, 1.f);
                    w[s] = moe_times(q, f);
                    wl[s] = moe_lost(q, f, w[s]);
                    const u32x4_t bits = __builtin_bit_cast(u32x4_t, wl[s]);
                    any |= (bits[0] | bits[1] | bits[2] | bits[3]) & 0x7FFF7FFFu;
                }
                lost = __ballot(any != 0u) != 0ull;
            } else if constexpr (MX) {
                const uint32_t e8 = row[17u * i];
                s0 = __uint_as_float(e8 ? e8 << 23 : 0x00400000u);  // 2^(e - 127)
                const float f = fold ? s0 : 1.f;
#pragma unroll
                for (int s = 0; s < 2; ++s) w[s] = moe_payload<TY>(row, i, 2u * s + h, f);
            } else {
#pragma unroll
                for (int s = 0; s < 2; ++s) w[s] = mms_operand<TY>(row, i, 2u * s + h, s0, s1);
            }
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
                if (tt == 0 || both) {
                    if (TY == 1 || KQ || fold) {
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int f = 0; f < HALVES; ++f) acc[tt][rt] = mul(x[f][tt][s], w[s], acc[tt][rt]);
                        if constexpr (Q6)
                            if (lost) {
#pragma unroll
                                for (int s = 0; s < 2; ++s) acc[tt][rt] = mul(x[0][tt][s], wl[s], acc[tt][rt]);
                            }
                    } else {
                        moe_f32x16 d = {};
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int f = 0; f < HALVES; ++f) d = mul(x[f][tt][s], w[s], d);
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[tt][rt][j] = fmaf(s0, d[j], acc[tt][rt][j]);
                    }
                }
        }
    };
    // the accumulators from the last super-block's unit to this one's
    auto rescale = [&]() {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const uint8_t *row = wbuf[wave] + (32u * rt + n) * F::RS;
            const float d = mms_f16(*(const uint16_t *) (row + (Q6 ? 208u + MmsFmt<14>::LAST : 0u)));
            counts[rt] = d != 0.f;
            const float ratio = counts[rt] ? unit[rt] / d : 1.f;
            unit[rt] = counts[rt] ? d : unit[rt];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[tt][rt][j] *= ratio;
        }
    };
    auto mins = [&]() {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const u32x4_t hd = *(const u32x4_t *) (wbuf[wave] + (32u * rt + n) * F::RS);
            const float f = -mms_f16(hd[0] >> 16) / unit[rt];
            moe_bf8 m;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) m[k] = (__bf16) (float) moe_k4_min(hd, k);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
                if (tt == 0 || both) {
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

    uint32_t piece[2] = {0u, 0u};
    wload(0u);
    xload(0u);
    xput(0u);
    if constexpr (Q45) xsums(piece);
    xload(min(1u, total - 1u));
    moe_barrier();
    uint32_t step = 0;
    // The steps of a window. Sums: the pair that is stored for the next step has its own stored with it, but
    // the next window's first pair waits for that window, when the mins of this one have been taken.
    auto steps = [&](uint32_t skip) {
#pragma unroll
        for (uint32_t j = 0; j < SPW; ++j, ++step) {
            const uint32_t buf = step & 1u;
            if constexpr (Q45)
                if (j == 0) sput(piece, 0u);
            xput(buf ^ 1u);  // the pair after this one (after the last: nothing reads it)
            if constexpr (Q45) {
                xsums(piece);
                if (j + 1u < SPW) sput(piece, j + 1u);
            }
            xload(min(step + 2u, total - 1u));
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
                if (2u * j + b >= skip) compute(buf, b, 2u * j + b);
            if constexpr (Q45)
                if (j + 1u == SPW) mins();
            moe_barrier();
        }
    };
    for (uint32_t w = 0; w < n_win; ++w) {
        __builtin_amdgcn_wave_barrier();
        wput();
        __builtin_amdgcn_wave_barrier();
        wload(min(w + 1u, n_win - 1u));
        const uint32_t skip = w * WB - wstart(w);
        if constexpr (KQ) rescale();
        if constexpr (MX) {
            uint32_t lo = 255u, hi = 0u;  // of row `lane`
#pragma unroll
            for (uint32_t i = 0; i < WB; ++i) {
                const uint32_t e8 = wbuf[wave][lane * F::RS + 17u * i];
                lo = min(lo, e8);
                hi = max(hi, e8);
            }
            fold = __ballot(lo < 114u || hi > 139u) == 0ull;
        }
        steps(skip);
    }
    if constexpr (KQ) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[tt][rt][j] *= unit[rt];
    }

#pragma unroll
    for (int rt = 0; rt < (GU ? 1 : 2); ++rt) {
        const uint32_t r = r0 + 32u * rt + n;
        if (r >= a.rows) continue;
        const float b0 = a.bias[0] ? a.bias[0][(uint64_t) e * a.rows + r] : 0.f;
        const float b1 = GU && a.bias[1] ? a.bias[1][(uint64_t) e * a.rows + r] : 0.f;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t u = 32u * tt + 8u * (j >> 2) + 4u * h + (j & 3);
                if (u >= count) continue;
                const uint64_t o = (uint64_t) slots[u] * a.rows + r;
                if constexpr (GU) {
                    const float v = moe_activation(a, acc[tt][0][j] + b0, acc[tt][1][j] + b1);
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

}  // namespace

#define MOE_TILE(NAME, TY)                                                                                      \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))                \
    moearc_moe_tile_##NAME##_gu_f32_k(MoeArgs a) { moe_tile_body<TY, true, 2>(a); }                             \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))                \
    moearc_moe_tile_##NAME##_gu_f16_k(MoeArgs a) { moe_tile_body<TY, true, 1>(a); }                             \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))                \
    moearc_moe_tile_##NAME##_p_f32_k(MoeArgs a) { moe_tile_body<TY, false, 2>(a); }                             \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))                \
    moearc_moe_tile_##NAME##_p_f16_k(MoeArgs a) { moe_tile_body<TY, false, 1>(a); }
MOE_TILE(f16, 1)
MOE_TILE(q8_0, 8)
MOE_TILE(q4_k, 12)
MOE_TILE(q5_k, 13)
MOE_TILE(q6_k, 14)
MOE_TILE(mxfp4, 39)
