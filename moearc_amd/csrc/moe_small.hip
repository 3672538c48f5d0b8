// The experts' products for few slots per expert (MoeArgs): y[s][r] = sum_c W_e[r][c] x[s / x_div][c]
// (+ bias_e[r]) for the slots s of expert e, or, with two matrices, the activation of both products.
// Meant to be bound by reading the chosen experts' weights once.
//
// Work-group: 32 weight rows (16 of each of two matrices) of one expert and up to 16 of its slots at a
// time; its 8 waves cut the reduction between them and meet once, in LDS, at the end. A wave moves
// windows of its rows' bytes through registers and LDS (the next window in flight while the current one
// is multiplied) and reads MFMA operands from there, as matmul_small.hip does: lane (q, n) holds
// k 8q .. 8q + 7 of weight row n (B operand of v_mfma_f32_16x16x32_f16) and of token n (A operand).
// The launch has at most 64 slots: each wave finds its expert's from the ids by ballots, which saves a
// decode step a launch. Grid y is the slot; the work-groups of slots that are not their expert's first
// leave at once. Measured: 8 tokens of 4 of 64 Q5_K experts, 2048 x 2048, 14 to 22 of them woken (41 to 64 MB), 24 to
// 34 us, 1.7 to 1.9 TB/s: eight waves leave 2048 columns one window each, with nothing in flight behind it.
//
// f32 activations enter as f16 hi + lo (x = hi + lo to 2^-22 |x| or 2^-25), f16 ones as they are; weight payloads
// as exact f16 integers (E2M1 code points for MXFP4), each block's f32 sum scaled in f32.
#include "common.h"

namespace {

// As MmsFmt, with windows short enough that 8 waves of two 16-row groups leave LDS for several work-groups.
template <uint32_t TY>
struct MoeFmt {
    static constexpr uint32_t WB = TY == 1 ? 2 : TY == 8 ? 4 : 8;
    static constexpr uint32_t S = WB * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
    static constexpr uint32_t NP = (S + 15u) / 16u, NI = (NP + 3u) / 4u;
    static constexpr uint32_t RS = 16u * NP + (NP % 2u ? 0u : 16u);
    // Q8_0: 136 bytes, the last piece goes where its bytes belong (8-byte aligned), in two halves
    static constexpr bool SPLIT_LAST = TY == 8;
};

// min and max that hand a NaN on (fminf and fmaxf drop it, and a token whose gate is NaN would come out as the limit). As
// instructions: the build leaves the compiler free to take a NaN for impossible.
__device__ __forceinline__ float moe_min(float a, float b) {
    float r;
    asm("v_minimum3_f32 %0, %1, %2, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float moe_max(float a, float b) {
    float r;
    asm("v_maximum3_f32 %0, %1, %2, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

template <typename Args>
__device__ __forceinline__ float moe_activation(const Args &a, float g, float u) {
    // exp2 of a large positive argument is +inf and g / inf is 0: no branch needed
    if (a.clamped) {
        g = moe_min(g, a.limit);
        u = moe_min(moe_max(u, -a.limit), a.limit);
        return g / (1.f + expf(-a.alpha * g)) * (u + 1.f);
    }
    return g / (1.f + expf(-g)) * u;
}

template <uint32_t TY, bool GU, bool XH>
__device__ __forceinline__ void moe_small_body(const MoeArgs &a) {
    using F = MoeFmt<TY>;
    constexpr uint32_t WB = F::WB, W = MOEARC_MOE_SMALL_WAVES, CK = WB >= 4 ? 2 : 1;
    constexpr bool Q45 = TY == 12 || TY == 13;
    static_assert(WB % (2 * CK) == 0, "activation batches alternate within a window");
    __shared__ __attribute__((aligned(16))) uint8_t wlds[W][2][16 * F::RS];
    __shared__ u32x4_t xlds[W][2][64];  // a k-block's activations in f16 (hi, lo); at the end the sums
    __shared__ uint32_t slots[64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 15u, lq = lane >> 4;

    // the expert and its slots
    uint32_t e, count;
    const uint32_t id = lane < a.n_slots ? a.ids[lane] : MOEARC_NO_EXPERT;
    e = __builtin_amdgcn_readlane(id, blockIdx.y);
    if (e >= a.n_expert) {
        if (e != MOEARC_NO_EXPERT && blockIdx.x == 0u && tid == 0u) *(volatile uint32_t *) a.err = 1u;
        e = a.n_expert;
        count = 1u;
        if (tid == 0u) slots[0] = blockIdx.y;
    } else {
        const uint64_t mask = __ballot(id == e);
        if (mask & ((1ull << blockIdx.y) - 1ull)) return;  // an earlier slot's work-groups have it
        count = (uint32_t) __popcll(mask);
        if (tid < 64u && id == e) slots[__popcll(mask & ((1ull << lane) - 1ull))] = lane;
    }
    const uint32_t rbase = (GU ? 16u : 32u) * blockIdx.x;
    if (e == a.n_expert) {  // no expert: no product
        if (!GU && a.zero_skipped) {
            __syncthreads();
            for (uint32_t i = tid; i < 32u * count; i += 64u * W) {
                const uint32_t r = rbase + (i & 31u);
                const uint64_t o = (uint64_t) slots[i >> 5] * a.rows + r;
                if (r >= a.rows) continue;
                if (a.y_f16) ((uint16_t *) a.y)[o] = 0;
                else ((float *) a.y)[o] = 0.f;
            }
        }
        return;
    }
    __syncthreads();

    const uint32_t nb_all = a.cols / 32u, kb0 = min(wave * a.kb_per, nb_all), end = min(kb0 + a.kb_per, nb_all);
    // group g's rows: matrix g's (gate, up), or the next 16 of the one matrix
    const uint8_t *wsrc[2];
#pragma unroll
    for (uint32_t g = 0; g < 2; ++g)
        wsrc[g] = a.w[GU ? g : 0] + e * a.expert_bytes +
                  (uint64_t) min(rbase + (GU ? 0u : 16u * g) + (lane >> 2), a.rows - 1u) * a.row_bytes;
    u32x4_t wreg[2][F::NI];
    auto wload = [&](uint32_t b) {  // the window that starts at block b
        const uint64_t o = (uint64_t) b * 32u / moearc_mv_be(TY) * moearc_mv_bb(TY);
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
#pragma unroll
            for (uint32_t j = 0; j < F::NI; ++j)
                __builtin_memcpy(&wreg[g][j], wsrc[g] + o + min(16u * (4u * j + (lane & 3u)), F::S - 16u), 16);
    };
    auto wput = [&]() {
#pragma unroll
        for (uint32_t g = 0; g < 2; ++g)
#pragma unroll
            for (uint32_t j = 0; j < F::NI; ++j) {
                uint8_t *row = wlds[wave][g] + F::RS * (lane >> 2);
                const uint32_t p = min(4u * j + (lane & 3u), F::NP - 1u);
                if constexpr (F::SPLIT_LAST) {
                    const uint32_t o = min(16u * p, F::S - 16u);
                    *(u32x2_t *) (row + o) = u32x2_t{wreg[g][j][0], wreg[g][j][1]};
                    *(u32x2_t *) (row + o + 8u) = u32x2_t{wreg[g][j][2], wreg[g][j][3]};
                } else {
                    *(u32x4_t *) (row + 16u * p) = wreg[g][j];
                }
            }
    };
    for (uint32_t t0 = 0; t0 < count; t0 += MOEARC_MOE_SMALL_TOKENS) {
        const uint32_t here = min(count - t0, MOEARC_MOE_SMALL_TOKENS);
        // f32: load i, lane l: token 8 i + l / 8, floats 4 (l % 8) .. + 3 of the block; f16: token l / 4,
        // halves 8 (l % 4) .. + 7. Lanes of absent tokens load nothing and hold zeros.
        constexpr int NX = XH ? 1 : 2;
        const uint8_t *x[NX];
        bool live[NX];
        uint32_t put[2], get;
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            const uint32_t u = XH ? lane >> 2 : 8u * i + (lane >> 3);
            live[i] = u < here;
            const uint64_t row = slots[t0 + min(u, here - 1u)] / a.x_div;
            x[i] = (const uint8_t *) a.x + (row * a.cols) * (XH ? 2u : 4u) + 16u * (XH ? lane & 3u : lane & 7u);
            const uint32_t c = lane & 7u;
            put[i] = XH ? 4u * u + ((lane & 3u) ^ (u >> 2)) : 2u * (4u * u + ((c >> 1) ^ (u >> 2))) + (c & 1u);
        }
        // token u's 16-byte slot q (k 8 q .. + 7) is at q ^ (u / 4). f32: row 4 q + k of the A operand, and
        // of D, is token mms_token(q, k), whose block sums are in the lanes that D's lanes can reach by DPP;
        // f16: row and token are the same.
        const uint32_t un = XH ? n : mms_token(n >> 2, n & 3u);
        get = 4u * un + (lq ^ (un >> 2));
        struct Batch {
            u32x4_t x[CK][NX];
        };
        auto xload = [&](Batch &o, uint32_t b0) {
#pragma unroll
            for (uint32_t i = 0; i < CK; ++i) {
                const uint64_t b = (uint64_t) min(b0 + i, nb_all - 1u) * (XH ? 64u : 128u);
#pragma unroll
                for (int k = 0; k < NX; ++k) {
                    o.x[i][k] = u32x4_t{0u, 0u, 0u, 0u};
                    if (live[k]) __builtin_memcpy(&o.x[i][k], x[k] + b, 16);
                }
            }
        };
        float4_t acc[2];
        acc[0] = acc[1] = float4_t{0.f, 0.f, 0.f, 0.f};
        const float4_t zero = {0.f, 0.f, 0.f, 0.f};
        auto compute = [&](const Batch &o, uint32_t ws, uint32_t i0, uint32_t lo_b) {
#pragma unroll
            for (uint32_t i = 0; i < CK; ++i) {
                const uint32_t b = ws + i0 + i;
                if (b < lo_b || b >= end) continue;  // uniform
                float sum[NX];
                __builtin_amdgcn_wave_barrier();
                if constexpr (XH) {
                    xlds[wave][0][put[0]] = o.x[i][0];
                    if constexpr (Q45) {  // the block sum of token lane / 4, over its four lanes
                        float s = 0.f;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t pair = o.x[i][0][k];  // a copy: bit_cast of an element takes element 0
                            const half2_t h = __builtin_bit_cast(half2_t, pair);
                            s += (float) h[0] + (float) h[1];
                        }
                        s += dpp<0xB1>(s);
                        sum[0] = s + dpp<0x4E>(s);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < NX; ++k) {
                        const float4_t v = __builtin_bit_cast(float4_t, o.x[i][k]);
                        mms_half4 hi, lo;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            hi[c] = (_Float16) v[c];
                            lo[c] = (_Float16) (v[c] - (float) hi[c]);
                        }
                        ((mms_half4 *) xlds[wave][0])[put[k]] = hi;
                        ((mms_half4 *) xlds[wave][1])[put[k]] = lo;
                        if constexpr (Q45) {  // of token 8 k + lane / 8, over its eight lanes
                            float s = (v[0] + v[1]) + (v[2] + v[3]);
                            s += dpp<0xB1>(s);
                            s += dpp<0x4E>(s);
                            sum[k] = s + dpp<0x141>(s);
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
                const half8_t hi = __builtin_bit_cast(half8_t, xlds[wave][0][get]);
                half8_t lo = {};
                if constexpr (!XH) lo = __builtin_bit_cast(half8_t, xlds[wave][1][get]);
                auto mul = [&](half8_t w, float4_t c) {
                    c = mms_mfma(hi, w, c);
                    if constexpr (!XH) c = mms_mfma(lo, w, c);
                    return c;
                };
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float s0, s1;
                    const half8_t bw = mms_operand<TY>(wlds[wave][g] + F::RS * n, i0 + i, lq, s0, s1);
                    if constexpr (TY == 1) {
                        acc[g] = mul(bw, acc[g]);
                    } else if constexpr (TY == 14) {  // the two 16-wide scale groups: k 0 .. 15 and 16 .. 31
                        const half8_t none = {};
                        const float4_t d0 = mul(lq < 2u ? bw : none, zero), d1 = mul(lq < 2u ? none : bw, zero);
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[g][k] = fmaf(s1, d1[k], fmaf(s0, d0[k], acc[g][k]));
                    } else {
                        const float4_t d = mul(bw, zero);
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[g][k] = fmaf(s0, d[k], acc[g][k]);
                        if constexpr (Q45) {
                            if constexpr (XH) {  // D's rows 4 lq + k: the tokens of this lane's 16 lanes
                                acc[g][0] = fmaf(dpp<0x150>(sum[0]), -s1, acc[g][0]);
                                acc[g][1] = fmaf(dpp<0x154>(sum[0]), -s1, acc[g][1]);
                                acc[g][2] = fmaf(dpp<0x158>(sum[0]), -s1, acc[g][2]);
                                acc[g][3] = fmaf(dpp<0x15C>(sum[0]), -s1, acc[g][3]);
                            } else {
                                acc[g][0] = fmaf(dpp<0x150>(sum[0]), -s1, acc[g][0]);
                                acc[g][1] = fmaf(dpp<0x158>(sum[0]), -s1, acc[g][1]);
                                acc[g][2] = fmaf(dpp<0x150>(sum[1]), -s1, acc[g][2]);
                                acc[g][3] = fmaf(dpp<0x158>(sum[1]), -s1, acc[g][3]);
                            }
                        }
                    }
                }
            }
        };
        if (kb0 < end) {
            // windows of WB blocks from kb0; one that would pass the row's end starts earlier, its first
            // blocks skipped (the host sends rows of at least WB blocks)
            Batch p, q;
            uint32_t ws = min(kb0, nb_all - WB);
            wload(ws);
            xload(p, ws);
            for (uint32_t b = kb0; b < end; b += WB) {
                const uint32_t next = min(b + WB, nb_all - WB);
                __builtin_amdgcn_wave_barrier();
                wput();
                __builtin_amdgcn_wave_barrier();
                wload(next);
#pragma unroll
                for (uint32_t i = 0; i < WB; i += 2 * CK) {
                    xload(q, ws + i + CK);
                    compute(p, ws, i, b);
                    xload(p, i + 2 * CK < WB ? ws + i + 2 * CK : next);
                    compute(q, ws, i + CK, b);
                }
                ws = next;
            }
        }
        __builtin_amdgcn_wave_barrier();
        float *red = (float *) xlds[wave];  // [group][token][row]
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) red[256u * g + 16u * (XH ? 4u * lq + k : mms_token(lq, k)) + n] = acc[g][k];
        __syncthreads();
        // output i: token i / R, row i % R, the waves' sums in order
        constexpr uint32_t R = GU ? 16u : 32u;
        for (uint32_t i = tid; i < 16u * R; i += 64u * W) {
            const uint32_t u = i / R, rl = i % R, r = rbase + rl;
            float s[GU ? 2 : 1];
#pragma unroll
            for (uint32_t g = 0; g < (GU ? 2u : 1u); ++g) {
                const uint32_t at = GU ? 256u * g + 16u * u + rl : 256u * (rl >> 4) + 16u * u + (rl & 15u);
                s[g] = ((const float *) xlds[0])[at];
#pragma unroll
                for (uint32_t w = 1; w < W; ++w) s[g] += ((const float *) xlds[w])[at];
            }
            if (u < here && r < a.rows) {
                const uint64_t o = (uint64_t) slots[t0 + u] * a.rows + r;
#pragma unroll
                for (uint32_t g = 0; g < (GU ? 2u : 1u); ++g)
                    if (a.bias[g]) s[g] += a.bias[g][(uint64_t) e * a.rows + r];
                float v;
                if constexpr (GU) v = moe_activation(a, s[0], s[1]);
                else v = s[0];
                if (a.y_f16) ((_Float16 *) a.y)[o] = (_Float16) v;
                else ((float *) a.y)[o] = v;
            }
        }
        __syncthreads();
    }
}

}  // namespace

#define MOE_SMALL(NAME, TY)                                                                                       \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MOE_SMALL_WAVES, 4) moearc_moe_small_##NAME##_gu_f32_k(MoeArgs a) { \
        moe_small_body<TY, true, false>(a);                                                                       \
    }                                                                                                             \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MOE_SMALL_WAVES, 4) moearc_moe_small_##NAME##_gu_f16_k(MoeArgs a) { \
        moe_small_body<TY, true, true>(a);                                                                        \
    }                                                                                                             \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MOE_SMALL_WAVES, 4) moearc_moe_small_##NAME##_p_f32_k(MoeArgs a) { \
        moe_small_body<TY, false, false>(a);                                                                      \
    }                                                                                                             \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MOE_SMALL_WAVES, 4) moearc_moe_small_##NAME##_p_f16_k(MoeArgs a) { \
        moe_small_body<TY, false, true>(a);                                                                       \
    }
MOE_SMALL(f16, 1)
MOE_SMALL(q8_0, 8)
MOE_SMALL(q4_k, 12)
MOE_SMALL(q5_k, 13)
MOE_SMALL(q6_k, 14)
MOE_SMALL(mxfp4, 39)
