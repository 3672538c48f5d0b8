// The experts' products for a single token, the decode step: bound by reading the chosen experts' weights, and
// short enough for the launches' latency to count, so two launches do it all:
//   gate_up: act[j][r] = act(W_gate[e_j] x + b, W_up[e_j] x + b), e_j = ids[j]
//   down:    y[r] (+)= sum over j of weights[j] (W_down[e_j] act[j] + b)
// Matrix-vector products as matvec.hip makes them (its formats' dot products): a lane owns the pieces lane, lane
// + 64, ... of every row and holds the inputs of its pieces in registers; rows come through LDS, two in flight per
// wave. A wave's units here are gate and up of one row in turn, whose results meet in it, or the rows of one
// expert after the other, summed in the order of j: no wave waits for another, and nothing is added in memory.
// Measured: four MXFP4 experts of 2880 x 2880 in 14.0 us (gate and up, 35 MB) and 13.2 (down, 18 MB: one row a wave, and
// every work-group stages the four inputs), against 44 for both as products of moe_small.hip with their sum in a launch
// of its own.
#include "common.h"

extern __shared__ __attribute__((aligned(16))) uint8_t mvx_smem[];

namespace {

template <uint32_t TY, uint32_t PPL, bool GU>
__device__ __forceinline__ void moe_vec_body(const MoeVecArgs &a) {
    constexpr uint32_t BB = moearc_mv_bb(TY), BE = moearc_mv_be(TY), PE = Fmt<TY>::PE;
    constexpr uint32_t PPB = BE >= PE ? BE / PE : 1u;  // pieces per block
    constexpr uint32_t GMAX = moearc_mv_gmax(TY, PPL);
    constexpr uint32_t XPAD = PE + 4u;                 // LDS floats per piece of an input row
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t P = a.n_pieces;
    const uint32_t r0 = (blockIdx.x * waves + wave) * a.rpw, n_rows = r0 < a.rows ? min(a.rpw, a.rows - r0) : 0u;

    // the experts: lane j holds the j-th id; GU: this work-group's, else those that count, in order
    const uint32_t id = lane < a.n_used ? a.ids[lane] : MOEARC_NO_EXPERT;
    const uint64_t valid = __ballot(id < a.n_expert);
    uint32_t n_slots = 1u;
    if constexpr (GU) {
        if (blockIdx.x == 0u && blockIdx.y == 0u && wave == 0u && id >= a.n_expert && id != MOEARC_NO_EXPERT)
            *(volatile uint32_t *) a.err = 1u;  // (down would say the same)
        if (!((valid >> blockIdx.y) & 1ull)) return;
    } else {
        n_slots = (uint32_t) __popcll(valid);
    }
    auto slot_of = [&](uint32_t q) -> uint32_t {  // the q-th slot that counts
        if constexpr (GU) return blockIdx.y;
        uint64_t m = valid;
        for (uint32_t i = 0; i < q; ++i) m &= m - 1ull;
        return (uint32_t) __builtin_ctzll(m);
    };
    const uint32_t per_slot = GU ? 2u * n_rows : n_rows, units = n_slots * per_slot;

    uint8_t *wb = mvx_smem + a.x_lds_bytes + wave * a.wave_buf;
    const uint32_t wb_off = a.x_lds_bytes + wave * a.wave_buf;
    auto piece_byte = [&](uint32_t p) -> uint32_t { return BE == 1u ? p * (PE * BB) : (p / PPB) * BB; };

    u32x4_t ga[GMAX], gb[GMAX];
    uint32_t da = 0, na = 0, db = 0, nb = 0;  // LDS offset of the row's first byte, 16-byte granules of the row
    auto issue = [&](uint32_t u, u32x4_t (&g)[GMAX], uint32_t &delta, uint32_t &ng) {
        const uint32_t q = u / per_slot, i = u % per_slot, s = slot_of(q);
        const uint32_t e = __builtin_amdgcn_readlane(id, s);
        const uint32_t r = r0 + (GU ? i >> 1 : i);
        const uint8_t *W = GU && (i & 1u) ? a.w[1] : a.w[0];
        const uintptr_t src = (uintptr_t) (W + e * a.expert_bytes + (uint64_t) r * a.row_bytes), base = src & ~(uintptr_t) 15;
        delta = (uint32_t) (src - base);
        ng = (uint32_t) ((delta + a.row_bytes + 15u) >> 4);
#pragma unroll
        for (uint32_t k = 0; k < GMAX; ++k) g[k] = gload16(base + 16u * (uintptr_t) min(lane + 64u * k, ng - 1u));
    };
    if (units) {  // the first rows are on their way before anything waits for the inputs
        issue(0u, ga, da, na);
        issue(min(1u, units - 1u), gb, db, nb);
    }
    // what goes to each result: GU: lane i: bias of row i / 2, matrix i % 2; else lane q * n_rows + i: of slot q, row i
    float bias = 0.f, weight = 0.f, old = 0.f;
    if constexpr (GU) {
        const uint32_t e = __builtin_amdgcn_readlane(id, blockIdx.y);
        const float *b = lane & 1u ? a.bias[1] : a.bias[0];
        if (b && lane < 2u * n_rows) bias = b[(uint64_t) e * a.rows + r0 + (lane >> 1)];
    } else {
        if (lane < a.n_used && ((valid >> lane) & 1ull)) weight = a.weights[lane];
        if (units) {  // (uniform: every lane takes part in the exchange)
            const uint32_t e = (uint32_t) __shfl((int) id, (int) slot_of(min(lane / n_rows, n_slots - 1u)));
            if (a.bias[0] && lane < units) bias = a.bias[0][(uint64_t) e * a.rows + r0 + lane % n_rows];
        }
        if (a.accumulate && lane < n_rows) old = ((const float *) a.y)[r0 + lane];
    }
    // the inputs, f32, piece p of a row at floats [p * XPAD, + PE): one row, or the slots' that count
    {
        float *xl = (float *) mvx_smem;
        const uint32_t quads = a.n_pieces * (PE / 4u), n = n_slots * quads;  // four floats at a time, of all rows
        for (uint32_t c0 = threadIdx.x; c0 < n; c0 += 8u * blockDim.x) {
            float v[8][4];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t i = min(c0 + k * blockDim.x, n - 1u), q = GU ? 0u : i / quads;
                const uint64_t at = (GU ? 0ull : (uint64_t) slot_of(q) * a.cols) + min(4u * (i - q * quads), a.cols - 4u);
                if (a.x_f16) {
                    _Float16 h[4];
                    __builtin_memcpy(h, (const _Float16 *) a.x + at, 8);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k][j] = (float) h[j];
                } else {
                    __builtin_memcpy(v[k], (const float *) a.x + at, 16);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t i = c0 + k * blockDim.x, q = GU ? 0u : i / quads, c = 4u * (i - q * quads);
                if (i < n) *(float4_t *) (xl + q * P * XPAD + (c / PE) * XPAD + c % PE) = c < a.cols ? float4_t{v[k][0], v[k][1], v[k][2], v[k][3]} : float4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
        __syncthreads();
    }
    if (!units) {
        if constexpr (!GU)  // no expert at all: the sum is empty
            if (!a.accumulate && lane < n_rows) {
                if (a.y_f16) ((_Float16 *) a.y)[r0 + lane] = (_Float16) 0.f;
                else ((float *) a.y)[r0 + lane] = 0.f;
            }
        return;
    }
    float xr[PPL][PE], xs[PPL];
    auto load_x = [&](uint32_t q) {
#pragma unroll
        for (uint32_t i = 0; i < PPL; ++i) {
            const float *xl = (const float *) mvx_smem + (uint64_t) (q * P + min(lane + 64u * i, P - 1u)) * XPAD;
            float t = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < PE; j += 4) {
                const float4_t v = *(const float4_t *) (xl + j);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    xr[i][j + k] = v[k];
                    if constexpr (needs_xsum(TY)) t += v[k];
                }
            }
            xs[i] = t;
        }
    };
    float sum = 0.f, gate = 0.f;  // of row r0 + lane; GU: the gate's product, until the up's arrives
    auto step = [&](uint32_t u, u32x4_t (&g)[GMAX], uint32_t &delta_ref, uint32_t &ng_ref) {
        const uint32_t q = u / per_slot, i = u % per_slot, delta = delta_ref, ng = ng_ref;
#pragma unroll
        for (uint32_t k = 0; k < GMAX; ++k)
            if (lane + 64u * k < ng) *(u32x4_t *) (wb + 16u * (lane + 64u * k)) = g[k];
        issue(min(u + 2u, units - 1u), g, delta_ref, ng_ref);
        __builtin_amdgcn_wave_barrier();
        if (GU ? u == 0u : i == 0u) load_x(q);
        float acc = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < PPL; ++k) {
            const uint32_t p = lane + 64u * k;
            if (p < P) acc = Fmt<TY>::dot(mvx_smem, wb_off + delta + piece_byte(p), p % PPB, xr[k], xs[k], acc, BE == 1u ? min(PE, a.cols - p * PE) : PE);
        }
        __builtin_amdgcn_wave_barrier();
        acc = wave_sum_to_lane63(acc);
        float tot = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(acc), 63));
        tot += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(bias), GU ? i : u));
        if constexpr (GU) {
            if (i & 1u) {
                if (lane == (i >> 1)) sum = tot;  // up; the gate's is in `gate` of the same lane
            } else if (lane == (i >> 1)) {
                gate = tot;
            }
        } else {
            const float wt = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), slot_of(q)));
            if (lane == i) sum = fmaf(wt, tot, sum);
        }
    };
    for (uint32_t u = 0; u < units; u += 2u) {
        step(u, ga, da, na);
        if (u + 1u < units) step(u + 1u, gb, db, nb);
    }
    if (lane < n_rows) {
        float v;
        if constexpr (GU) v = moe_activation(a, gate, sum);
        else v = a.accumulate ? old + sum : sum;
        const uint64_t o = (GU ? (uint64_t) blockIdx.y * a.rows : 0u) + r0 + lane;
        if (a.y_f16) ((_Float16 *) a.y)[o] = (_Float16) v;
        else ((float *) a.y)[o] = v;
    }
}

}  // namespace

#define MOE_VEC_KERNEL(NAME, TY, PPL)                                                                  \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MV_MAX_WAVES) moearc_moe_vec_##NAME##_gu_p##PPL##_k(MoeVecArgs a) { \
        moe_vec_body<TY, PPL, true>(a);                                                                \
    }                                                                                                  \
    extern "C" __global__ void __launch_bounds__(64 * MOEARC_MV_MAX_WAVES) moearc_moe_vec_##NAME##_down_p##PPL##_k(MoeVecArgs a) { \
        moe_vec_body<TY, PPL, false>(a);                                                               \
    }
#define MOE_VEC(NAME, TY)        \
    MOE_VEC_KERNEL(NAME, TY, 1)  \
    MOE_VEC_KERNEL(NAME, TY, 2)  \
    MOE_VEC_KERNEL(NAME, TY, 4)
MOE_VEC(f16, 1)
MOE_VEC(q8_0, 8)
MOE_VEC(q4_k, 12)
MOE_VEC(q5_k, 13)
MOE_VEC(q6_k, 14)
MOE_VEC(mxfp4, 39)
