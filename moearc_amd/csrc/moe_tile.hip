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

template <uint32_t TY, bool GU, int HALVES>
__device__ __forceinline__ void moe_tile_body(const MoeArgs &a) {
    using F = MoeTileFmt<TY>;
    constexpr uint32_t WB = F::WB, SPW = WB / 2u;
    constexpr bool Q45 = TY == 12 || TY == 13, Q6 = TY == 14;
    constexpr uint32_t XB = 4096u, XPAIR = 2u * HALVES * XB;  // one half of a k-block, a pair of k-blocks
    __shared__ __attribute__((aligned(1024))) uint8_t xbuf[2 * XPAIR];
    __shared__ __attribute__((aligned(16))) uint8_t wbuf[4][64 * F::RS];
    __shared__ uint32_t slots[64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 31u, h = lane >> 5;

    const uint32_t ti = blockIdx.x / a.row_tiles, rt_i = blockIdx.x % a.row_tiles;
    if (ti >= *a.n_tiles) return;
    const MoeTile t = a.tiles[ti];
    const uint32_t e = __builtin_amdgcn_readfirstlane(t.expert), count = __builtin_amdgcn_readfirstlane(t.count);
    if (tid < count) slots[tid] = a.list[t.first + tid];
    __syncthreads();
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

    moe_f32x16 acc[2][2];  // [slot half][row tile]
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[tt][rt][j] = 0.f;

    // Q4_K, Q5_K: the block's sum of each slot's inputs, for the mins, is computed beside the products: the
    // ones operand gives D[slot][*] = sum of the block
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
        moe_f32x16 sums[2];
        if constexpr (Q45) {
            half8_t ones;
#pragma unroll
            for (int k = 0; k < 8; ++k) ones[k] = (_Float16) 1.f;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
                if (tt == 0 || both) {
                    sums[tt] = moe_f32x16{};
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int f = 0; f < HALVES; ++f)
                            sums[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[f][tt][s], ones, sums[tt], 0, 0, 0);
                }
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const uint8_t *row = wbuf[wave] + (32u * rt + n) * F::RS;
            half8_t w[2];
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int s = 0; s < 2; ++s) w[s] = mms_operand<TY>(row, i, 2u * s + h, s0, s1);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
                if (tt == 0 || both) {
                    if constexpr (TY == 1) {
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int f = 0; f < HALVES; ++f)
                                acc[tt][rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[f][tt][s], w[s], acc[tt][rt], 0, 0, 0);
                    } else if constexpr (Q6) {  // slice s is a 16-wide scale group
                        moe_f32x16 d0 = {}, d1 = {};
#pragma unroll
                        for (int f = 0; f < HALVES; ++f) {
                            d0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[f][tt][0], w[0], d0, 0, 0, 0);
                            d1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[f][tt][1], w[1], d1, 0, 0, 0);
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[tt][rt][j] = fmaf(s1, d1[j], fmaf(s0, d0[j], acc[tt][rt][j]));
                    } else {
                        moe_f32x16 d = {};
#pragma unroll
                        for (int s = 0; s < 2; ++s)
#pragma unroll
                            for (int f = 0; f < HALVES; ++f)
                                d = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[f][tt][s], w[s], d, 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            acc[tt][rt][j] = fmaf(s0, d[j], acc[tt][rt][j]);
                            if constexpr (Q45) acc[tt][rt][j] = fmaf(-s1, sums[tt][j], acc[tt][rt][j]);
                        }
                    }
                }
        }
    };

    wload(0u);
    xload(0u);
    xput(0u);
    xload(min(1u, total - 1u));
    moe_barrier();
    uint32_t step = 0;
    for (uint32_t w = 0; w < n_win; ++w) {
        __builtin_amdgcn_wave_barrier();
        wput();
        __builtin_amdgcn_wave_barrier();
        wload(min(w + 1u, n_win - 1u));
        const uint32_t ws = wstart(w), skip = w * WB - ws;
#pragma unroll
        for (uint32_t j = 0; j < SPW; ++j, ++step) {
            const uint32_t buf = step & 1u;
            xput(buf ^ 1u);  // the pair after this one (after the last: nothing reads it)
            xload(min(step + 2u, total - 1u));
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
                if (2u * j + b >= skip) compute(buf, b, 2u * j + b);
            moe_barrier();
        }
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
