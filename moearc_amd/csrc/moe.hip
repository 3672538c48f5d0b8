// The router of a mixture-of-experts block, the grouping of its choices, and the sum over a token's
// experts. The products between them: moe_small.hip, moe_tile.hip.
#include "common.h"

namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
    return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, CTRL, 0xF, 0xF, true);
}
// Over the 16 lanes of a row, in every one of them.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, dpp_u32<0xB1>(v));
    v = max(v, dpp_u32<0x4E>(v));
    v = max(v, dpp_u32<0x141>(v));
    return max(v, dpp_u32<0x140>(v));
}
__device__ __forceinline__ uint32_t row_min(uint32_t v) {
    v = min(v, dpp_u32<0xB1>(v));
    v = min(v, dpp_u32<0x4E>(v));
    v = min(v, dpp_u32<0x141>(v));
    return min(v, dpp_u32<0x140>(v));
}
__device__ __forceinline__ float row_sum(float v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}

// Float order as unsigned order: larger float, larger key; -0 and +0 alike; NaN (told by its bits) 1,
// below -inf. 0 is left for an expert already chosen.
__device__ __forceinline__ uint32_t route_key(float f) {
    uint32_t b = __float_as_uint(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
    if (b == 0x80000000u) b = 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float route_value(uint32_t key) {  // NaN comes back as -inf
    if (key <= 1u) return -INFINITY;
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
// exp(v - m) with m the row's largest: 1 at the largest also when it is infinite
__device__ __forceinline__ float route_exp(float v, float m) { return v == m ? 1.f : expf(v - m); }

// Sixteen lanes per token, four tokens per wave; lane l holds logits l, l + 16, ... as keys. A round takes
// the largest key left and, among equals, the lowest expert, over the 16 lanes by DPP. Lane j % 16 keeps
// choice j. (One token per wave measures the same work four times: 64 lanes reduce no faster than 16.) Bound by
// the rounds' vector instructions: 16,384 tokens, 8 of 128 experts (9.4 MB) 7.9 us; one token, 4 of 128, 3.0 us.
template <int PER>
__device__ __forceinline__ void route_body(const RouteArgs &a) {
    constexpr uint32_t L = MOEARC_ROUTE_LANES;
    const uint32_t tok = blockIdx.x * (blockDim.x / L) + threadIdx.x / L, lane = threadIdx.x % L;
    const bool live = tok < a.n_tok;  // a row of lanes without a token runs along and stores nothing
    const float *src = a.logits + (uint64_t) min(tok, a.n_tok - 1u) * a.n_expert;
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t e = L * i + lane;
        key[i] = e < a.n_expert ? route_key(src[e]) : 0u;
    }
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max(top, key[i]);
    top = row_max(top);
    const float m = route_value(top);
    float all = 0.f;
    if (a.over_all) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > 1u) all += route_exp(route_value(key[i]), m);
        all = row_sum(all);
    }
    // choices 16 p .. 16 p + 15 in pass p, stored unscaled; the sum over the chosen is known after the last
    float chosen = 0.f;
    uint32_t *ids = a.ids + (uint64_t) tok * a.n_used;
    float *weights = a.weights + (uint64_t) tok * a.n_used;
    const bool one = a.n_used <= L;
    float w_keep = 0.f;
    for (uint32_t j0 = 0; j0 < a.n_used; j0 += L) {
        uint32_t my_id = 0u;
        float my_e = 0.f;
        const uint32_t n = min(L, a.n_used - j0);
        for (uint32_t j = 0; j < n; ++j) {
            uint32_t best = 0u;
#pragma unroll
            for (int i = 0; i < PER; ++i) best = max(best, key[i]);
            best = row_max(best);
            uint32_t id = 0xFFFFFFFFu;
#pragma unroll
            for (int i = PER - 1; i >= 0; --i) id = key[i] == best ? L * i + lane : id;
            id = row_min(id);
#pragma unroll
            for (int i = 0; i < PER; ++i) key[i] = L * i + lane == id ? 0u : key[i];
            if (lane == j) {
                my_id = id;
                my_e = best > 1u ? route_exp(route_value(best), m) : 0.f;
            }
        }
        if (m == -INFINITY) my_e = 0.f;  // every expert masked: no weights
        chosen += row_sum(my_e);
        w_keep = my_e;
        if (live && lane < n) {
            ids[j0 + lane] = my_id;
            if (!one) weights[j0 + lane] = my_e;
        }
    }
    const float total = a.over_all ? all : chosen;
    const float f = total > 0.f ? a.scale / total : 0.f;
    if (!live) return;
    if (one) {
        if (lane < a.n_used) weights[lane] = w_keep * f;
    } else {
        for (uint32_t j = lane; j < a.n_used; j += L) weights[j] *= f;  // each lane its own stores
    }
}

}  // namespace

#define ROUTE_KERNEL(PER)                                                                                      \
    extern "C" __global__ void __launch_bounds__(256) moearc_moe_route_p##PER##_k(RouteArgs a) { route_body<PER>(a); }
ROUTE_KERNEL(1)
ROUTE_KERNEL(2)
ROUTE_KERNEL(4)
ROUTE_KERNEL(8)
ROUTE_KERNEL(16)
ROUTE_KERNEL(32)
ROUTE_KERNEL(64)

namespace {

// The plan (MoePlanArgs). One work-group per expert, and one for the slots without: each counts every
// group's slots itself (integer adds in LDS, so the order of the adds does not matter), from which it knows
// its group's first place and first tile, and then collects its own slots in order: each wave its share of the
// slots, counted, then placed. No work-group waits for another, and the result does not depend on their order.
// The ids are read once, all loads in flight, and kept in LDS (8000 slots: 9 us, and 13 when they were read twice,
// with two barriers for every 1024).
__device__ __forceinline__ void moe_plan_body(const MoePlanArgs &a) {
    __shared__ uint16_t ids[MOEARC_MOE_CHUNK_SLOTS];
    __shared__ uint32_t count[MOEARC_MAX_EXPERTS + 1];
    __shared__ uint32_t wave_n[16], before[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, mine = blockIdx.x;
    for (uint32_t e = tid; e <= a.n_expert; e += 1024u) count[e] = 0u;
    if (tid < 2u) before[tid] = 0u;
    __syncthreads();
    bool wrong = false;
    for (uint32_t s0 = tid; s0 < a.n_slots; s0 += 8u * 1024u) {
        uint32_t id[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) id[k] = a.ids[min(s0 + 1024u * k, a.n_slots - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k)
            if (s0 + 1024u * k < a.n_slots) {
                wrong = wrong || (id[k] >= a.n_expert && id[k] != MOEARC_NO_EXPERT);
                const uint32_t e = min(id[k], a.n_expert);
                ids[s0 + 1024u * k] = (uint16_t) e;
                atomicAdd(&count[e], 1u);
            }
    }
    if (wrong && mine == 0u) *(volatile uint32_t *) a.err = 1u;  // every writer stores the same
    __syncthreads();
    uint32_t slots = 0u, tiles = 0u;
    for (uint32_t e = tid; e < mine; e += 1024u) {
        slots += count[e];
        tiles += (count[e] + a.tile - 1u) / a.tile;
    }
    if (slots) {
        atomicAdd(&before[0], slots);
        atomicAdd(&before[1], tiles);
    }
    // this wave's share of the slots, 64 at a time
    const uint32_t share = (a.n_slots + 1023u) / 1024u * 64u, from = min(wave * share, a.n_slots), to = min(from + share, a.n_slots);
    uint32_t hits = 0u;
    for (uint32_t s0 = from; s0 < to; s0 += 64u) hits += (uint32_t) __popcll(__ballot(s0 + lane < to && ids[s0 + lane] == mine));
    if (lane == 0u) wave_n[wave] = hits;
    __syncthreads();
    const uint32_t n = count[mine], first = before[0], tile0 = before[1], n_tiles = (n + a.tile - 1u) / a.tile;
    for (uint32_t i = tid; i < n_tiles; i += 1024u)
        a.tiles[tile0 + i] = MoeTile{mine, first + i * a.tile, (uint16_t) min(a.tile, n - i * a.tile), 0, (uint16_t) i, (uint16_t) n_tiles};
    if (mine == a.n_expert && tid == 0u) *a.n_tiles = tile0 + n_tiles;
    uint32_t at = first;
#pragma unroll
    for (uint32_t w = 0; w < 16u; ++w) at += w < wave ? wave_n[w] : 0u;
    for (uint32_t s0 = from; s0 < to; s0 += 64u) {
        const bool hit = s0 + lane < to && ids[s0 + lane] == mine;
        const uint64_t mask = __ballot(hit);
        if (hit) a.list[at + (uint32_t) __popcll(mask & ((1ull << lane) - 1ull))] = s0 + lane;
        at += (uint32_t) __popcll(mask);
    }
}

// x for moe_tile.hip: f16 (of f32: hi, and the remainder lo) in the order of the weights' type, eight elements,
// one chunk, per thread.
template <bool F32>
__device__ __forceinline__ void moe_prep_body(const MoePrepArgs &a, uint32_t block, uint32_t blocks) {
    for (uint64_t i = (uint64_t) block * 1024u + threadIdx.x; i < a.n / 8u; i += (uint64_t) blocks * 1024u) {
        const uint32_t c = (uint32_t) i & 3u;
        const uint64_t blk = (i >> 2) * 32u;
        // the chunk's elements: two runs of four, from k0 and k1
        const bool mx = a.type == 39u, kq = a.type == 12u || a.type == 13u || a.type == 14u;
        const uint32_t k0 = mx ? 8u * (c & 1u) + 4u * (c >> 1) : 8u * c, k1 = mx ? k0 + 16u : k0 + 4u;
        _Float16 vh[8], vl[8];
        if constexpr (F32) {
            float v[8];
            __builtin_memcpy(v, (const float *) a.x + blk + k0, 16);
            __builtin_memcpy(v + 4, (const float *) a.x + blk + k1, 16);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                vh[k] = (_Float16) v[k];
                vl[k] = (_Float16) (v[k] - (float) vh[k]);
            }
        } else {
            __builtin_memcpy(vh, (const _Float16 *) a.x + blk + k0, 8);
            __builtin_memcpy(vh + 4, (const _Float16 *) a.x + blk + k1, 8);
        }
        half8_t hi, lo;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int q = (p & 4) | ((p & 1) << 1) | ((p >> 1) & 1), m = (p >> 1) | ((p & 1) << 2);
            hi[p] = mx ? vh[m] : kq ? vh[q] : vh[p];
            if constexpr (F32) lo[p] = mx ? vl[m] : kq ? vl[q] : vl[p];
        }
        *(half8_t *) (a.hi + 8u * i) = hi;
        if constexpr (F32) *(half8_t *) (a.lo + 8u * i) = lo;
    }
}

}  // namespace

// The inputs' order does not depend on the plan, and both are short: one launch, the plan's work-groups first (8000
// slots and 1000 f16 rows of 2048: 10.1 us, 14 as two).
extern "C" __global__ void __launch_bounds__(1024) moearc_moe_plan_k(MoePlanArgs a) { moe_plan_body(a); }
extern "C" __global__ void __launch_bounds__(1024) moearc_moe_plan_f32_k(MoePlanArgs a) {
    if (blockIdx.x <= a.n_expert) moe_plan_body(a);
    else moe_prep_body<true>(a.prep, blockIdx.x - a.n_expert - 1u, gridDim.x - a.n_expert - 1u);
}
extern "C" __global__ void __launch_bounds__(1024) moearc_moe_plan_f16_k(MoePlanArgs a) {
    if (blockIdx.x <= a.n_expert) moe_plan_body(a);
    else moe_prep_body<false>(a.prep, blockIdx.x - a.n_expert - 1u, gridDim.x - a.n_expert - 1u);
}

// The sum over a token's experts, four columns per thread (rows are whole blocks of 32): bound by reading the slots'
// rows once (2000 tokens of 4 slots of 2880: 92 MB in 27 us).
extern "C" __global__ void __launch_bounds__(256) moearc_moe_combine_k(MoeCombineArgs a) {
    const uint32_t tok = blockIdx.y, c = 4u * (blockIdx.x * 256u + threadIdx.x);
    if (c >= a.cols) return;
    float4_t s = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t j = 0; j < a.n_used; ++j) {
        const uint64_t slot = (uint64_t) tok * a.n_used + j;
        if (a.ids[slot] >= a.n_expert) continue;  // its rows were not computed, its weight is not looked at
        const float w = a.weights[slot];
        const float4_t v = *(const float4_t *) (a.part + slot * a.cols + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = fmaf(w, v[k], s[k]);
    }
    const uint64_t o = (uint64_t) tok * a.cols + c;
    if (a.y_f16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) ((_Float16 *) a.y)[o + k] = (_Float16) s[k];
    } else {
        float *y = (float *) a.y + o;
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = a.accumulate ? y[k] + s[k] : s[k];
    }
}
