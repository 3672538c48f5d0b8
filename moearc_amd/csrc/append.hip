// New tokens of a ragged batch on their way to the attention: q and k normed head by head (optional) and
// rotated at their positions, q written for the attention, K and V into the pages that the sequences' block
// tables name. Token i of a sequence's n new ones sits at position p = n_kv - n + i:
//   x' = x / sqrt(mean(x^2) + eps) * w
//   pair j of n_rot / 2:  (x0 cos a - x1 sin a, x0 sin a + x1 cos a) * mscale
//   a = p f_j,  f_j = base^(-2j / n_rot) / factors[j], mixed between interpolation and extrapolation (YaRN)
// Angles are f64: f32 leaves p f_0 4e-3 radians off at position 65536. A turn is reduced to [-1/2, 1/2] in f64
// and its sine and cosine are f32, once per work-group and pair, through LDS; every head of the token uses them.
// Bound by HBM for chunks, by latency for a decode step. A head takes LPH lanes of eight channels, held as the two
// quads that rotate into each other, so a head's norm is a sum over neighbouring lanes and every access is 16
// bytes a lane (8 of f16). Work-groups are (token, group of 256 / LPH heads of q, k and v), or of three times as many
// heads where there are more of these than the device holds at once: a work-group's life is mostly latency.
// Measured on MI355X: a token of 80 heads of 64 takes 3.7 us, as long as any launch of one work-group does, 48 tokens of 40
// normed heads of 128 4.2; 2048 tokens of one product's rows, f32 in and f16 out, 11.8 for 63 MB (5.3 TB/s, part of it from the
// last-level cache); 3709 tokens with f16 rows and an f32 cache 27.2 for 106 MB (3.9 TB/s: an f16 quad is 8 bytes a load).
#include "common.h"

#define AP_MAX_PAIRS 128  // head_dim <= 256

namespace {

// Accesses by pointers that ap_pick chose: their address space does not follow from where they came.
#define AP_GLOBAL __attribute__((address_space(1)))

struct ApQuad {
    float v[4];
};

__device__ __forceinline__ ApQuad ap_load(const void *p, uint64_t i, bool half) {
    ApQuad r;
    if (half) {
        const u32x2_t w = *(const AP_GLOBAL u32x2_t *) ((const AP_GLOBAL uint16_t *) p + i);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t pair = w[k];  // a copy: bit_cast of a vector's element takes element 0
            const half2_t h = __builtin_bit_cast(half2_t, pair);
            r.v[2 * k] = (float) h[0];
            r.v[2 * k + 1] = (float) h[1];
        }
    } else {
        const float4_t f = *(const AP_GLOBAL float4_t *) ((const AP_GLOBAL float *) p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) r.v[k] = f[k];
    }
    return r;
}

__device__ __forceinline__ void ap_store(void *p, uint64_t i, bool half, const ApQuad &r) {
    if (half) {
        const half2_t a = {(_Float16) r.v[0], (_Float16) r.v[1]}, b = {(_Float16) r.v[2], (_Float16) r.v[3]};
        *(AP_GLOBAL u32x2_t *) ((AP_GLOBAL uint16_t *) p + i) = u32x2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    } else {
        *(AP_GLOBAL float4_t *) ((AP_GLOBAL float *) p + i) = float4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
    }
}

// The sequence of row t: how many of the later sequences begin at or before it.
__device__ __forceinline__ uint32_t ap_sequence(const QkvAppendArgs &a, uint32_t t) {
    uint32_t g = 0;
#pragma unroll
    for (uint32_t i = 1; i < MOEARC_BATCH_SEQS / 8; ++i) g += t >= a.row_begin[8 * i];
    uint32_t b = 8 * g;
#pragma unroll
    for (uint32_t i = 1; i < 8; ++i) b += t >= a.row_begin[8 * g + i];
    return b;
}

// (cos, sin) * mscale of pair j at position pos.
__device__ __forceinline__ float2_t ap_angle(const QkvAppendArgs &a, uint32_t j, uint32_t pos) {
    double f = exp2((double) j * a.log2_step);
    if (a.factors) f /= (double) a.factors[j];
    if (a.ext_factor != 0.f) {
        // f64 too: an error of the mix is one of the angle, p f times as large
        const double ramp = ((double) j - (double) a.corr_lo) / fmax(0.001, (double) a.corr_hi - (double) a.corr_lo);
        const double mix = (1.0 - fmin(1.0, fmax(0.0, ramp))) * (double) a.ext_factor;
        f *= (double) a.freq_scale * (1.0 - mix) + mix;
    } else {
        f *= (double) a.freq_scale;
    }
    const double turns = (double) pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float) (turns - rint(turns)), &s, &c);
    return float2_t{c * a.mscale, s * a.mscale};
}

// Where a row goes: its sequence's page of the position, or nothing (an id outside the pool, reported).
struct ApPlace {
    uint32_t pos;
    bool has_pos, has_page;
    uint64_t token;  // page * page_tokens + slot
};

__device__ __forceinline__ ApPlace ap_place(const QkvAppendArgs &a, uint32_t t) {
    const uint32_t b = ap_sequence(a, t);
    ApPlace r;
    r.pos = a.n_kv[b] - a.n_new[b] + (t - a.row_begin[b]);
    r.has_pos = (int32_t) r.pos >= 0;  // n_kv below n_new: the first rows have none
    r.has_page = false;
    r.token = 0;
    if (r.has_pos) {
        const uint32_t page = r.pos / a.page_tokens;
        const uint32_t id = a.block_tables[b * a.bt_stride + page];
        r.has_page = id < a.n_pages;
        r.token = (uint64_t) id * a.page_tokens + (r.pos - page * a.page_tokens);
    }
    return r;
}

// One of three arguments by a lane's kind. The values are loaded first (the asm keeps them apart): a choice among
// their addresses would make the compiler copy the whole argument block to scratch memory.
__device__ __forceinline__ uint64_t ap_pick(uint32_t kind, uint64_t q, uint64_t k, uint64_t v) {
    asm("" : "+s"(q), "+s"(k), "+s"(v));
    return kind == 0 ? q : kind == 1 ? k : v;
}

// The sum over a head's LPH neighbouring lanes, in each of them.
template <int LPH>
__device__ __forceinline__ float ap_sum(float s) {
    s += dpp<0xB1>(s);   // quad_perm [1,0,3,2]
    s += dpp<0x4E>(s);   // quad_perm [2,3,0,1]
    s += dpp<0x141>(s);  // row_half_mirror
    if constexpr (LPH >= 16) s += dpp<0x140>(s);  // row_mirror
    if constexpr (LPH >= 32) s += __shfl_xor(s, 16);
    return s;
}

// NH heads to a thread, 256 / LPH apart: their loads are in flight together.
template <int LPH, int NH>
__device__ __forceinline__ void ap_body(const QkvAppendArgs &a) {
    __shared__ float2_t trig[AP_MAX_PAIRS];
    constexpr uint32_t HEADS = 256 / LPH;
    const uint32_t t = a.row_off + blockIdx.x, u = threadIdx.x % LPH;
    const uint32_t D = a.head_dim, nq = a.n_heads, nk = a.n_kv_heads;
    const bool half = a.in_f16, turned = 8 * u < a.n_rot;
    const uint32_t c0 = turned && a.neox ? 4 * u : 8 * u, c1 = turned && a.neox ? a.n_rot / 2 + 4 * u : 8 * u + 4;
    uint32_t kind[NH], own[NH];  // q, k, v; the head among its kind's
    bool live[NH];
    ApQuad x0[NH] = {}, x1[NH] = {};
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        const uint32_t head = (blockIdx.y * NH + i) * HEADS + threadIdx.x / LPH;
        kind[i] = head < nq ? 0u : head < nq + nk ? 1u : 2u;
        own[i] = kind[i] == 0 ? head : kind[i] == 1 ? head - nq : head - nq - nk;
        live[i] = head < nq + 2 * nk && 8 * u < D;
        if (live[i]) {
            const void *src = (const void *) ap_pick(kind[i], (uint64_t) a.q, (uint64_t) a.k, (uint64_t) a.v);
            const uint64_t at = t * ap_pick(kind[i], a.q_stride, a.k_stride, a.v_stride) + (uint64_t) own[i] * D;
            x0[i] = ap_load(src, at + c0, half);
            x1[i] = ap_load(src, at + c1, half);
        }
    }
    const ApPlace place = ap_place(a, t);
    if (!place.has_pos) return;
    if (!place.has_page && threadIdx.x == 0) *(volatile uint32_t *) a.err = 1u;  // every writer stores the same value
    if (2 * threadIdx.x < a.n_rot) trig[threadIdx.x] = ap_angle(a, threadIdx.x, place.pos);
    __syncthreads();
    float2_t cs[4] = {};
    if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = trig[4 * u + i];
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
        ApQuad &y0 = x0[i], &y1 = x1[i];
        const float *w = (const float *) ap_pick(kind[i], (uint64_t) a.q_norm, (uint64_t) a.k_norm, 0);
        if (w) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) s = fmaf(y0.v[k], y0.v[k], fmaf(y1.v[k], y1.v[k], s));
            s = 1.f / sqrtf(ap_sum<LPH>(s) / (float) D + a.eps);
            if (live[i]) {
                const ApQuad w0 = ap_load(w, c0, false), w1 = ap_load(w, c1, false);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    y0.v[k] = y0.v[k] * s * w0.v[k];
                    y1.v[k] = y1.v[k] * s * w1.v[k];
                }
            }
        }
        if (kind[i] < 2 && turned) {
            if (a.neox) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float r0 = y0.v[k], r1 = y1.v[k];
                    y0.v[k] = r0 * cs[k][0] - r1 * cs[k][1];
                    y1.v[k] = r0 * cs[k][1] + r1 * cs[k][0];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float r0 = y0.v[2 * k], r1 = y0.v[2 * k + 1], r2 = y1.v[2 * k], r3 = y1.v[2 * k + 1];
                    y0.v[2 * k] = r0 * cs[k][0] - r1 * cs[k][1];
                    y0.v[2 * k + 1] = r0 * cs[k][1] + r1 * cs[k][0];
                    y1.v[2 * k] = r2 * cs[2 + k][0] - r3 * cs[2 + k][1];
                    y1.v[2 * k + 1] = r2 * cs[2 + k][1] + r3 * cs[2 + k][0];
                }
            }
        }
        if (live[i] && (kind[i] == 0 || place.has_page)) {
            void *dst = (void *) ap_pick(kind[i], (uint64_t) a.q_out, (uint64_t) a.k_pages, (uint64_t) a.v_pages);
            const bool q_half = a.q_f16 != 0u, kv_half = a.kv_f16 != 0u, to_half = kind[i] == 0 ? q_half : kv_half;
            const uint64_t at = (kind[i] == 0 ? (uint64_t) t * nq + own[i] : place.token * nk + own[i]) * D;
            ap_store(dst, at + c0, to_half, y0);
            ap_store(dst, at + c1, to_half, y1);
        }
    }
}

__device__ __forceinline__ float ap_load1(const void *p, uint64_t i, bool half) {
    return half ? (float) ((const AP_GLOBAL _Float16 *) p)[i] : ((const AP_GLOBAL float *) p)[i];
}
__device__ __forceinline__ void ap_store1(void *p, uint64_t i, bool half, float v) {
    if (half) ((AP_GLOBAL _Float16 *) p)[i] = (_Float16) v;
    else ((AP_GLOBAL float *) p)[i] = v;
}

// Any head_dim up to 256, any alignment: a wave to a head, up to two pairs a lane (a rotated pair, or two channels
// behind the rotated ones, the last perhaps alone).
__device__ __forceinline__ void ap_any_body(const QkvAppendArgs &a) {
    __shared__ float2_t trig[AP_MAX_PAIRS];
    const uint32_t t = a.row_off + blockIdx.x, lane = threadIdx.x & 63u;
    const uint32_t head = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t D = a.head_dim, nq = a.n_heads, nk = a.n_kv_heads, half_rot = a.n_rot / 2;
    const uint32_t kind = head < nq ? 0u : head < nq + nk ? 1u : 2u;
    const uint32_t own = kind == 0 ? head : kind == 1 ? head - nq : head - nq - nk;
    const bool live = head < nq + 2 * nk;
    const ApPlace place = ap_place(a, t);
    if (!place.has_pos) return;
    if (!place.has_page && threadIdx.x == 0) *(volatile uint32_t *) a.err = 1u;
    if (threadIdx.x < half_rot) trig[threadIdx.x] = ap_angle(a, threadIdx.x, place.pos);
    __syncthreads();
    if (!live) return;
    const void *src = (const void *) ap_pick(kind, (uint64_t) a.q, (uint64_t) a.k, (uint64_t) a.v);
    const uint64_t from = t * ap_pick(kind, a.q_stride, a.k_stride, a.v_stride) + (uint64_t) own * D;
    float x[2][2];
    uint32_t c[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t j = lane + 64 * i;
        const bool turned = j < half_rot;
        c[i][0] = turned && a.neox ? j : 2 * j;
        c[i][1] = turned && a.neox ? j + half_rot : 2 * j + 1;
#pragma unroll
        for (int k = 0; k < 2; ++k) x[i][k] = c[i][k] < D ? ap_load1(src, from + c[i][k], a.in_f16) : 0.f;
    }
    const float *w = (const float *) ap_pick(kind, (uint64_t) a.q_norm, (uint64_t) a.k_norm, 0);
    if (w) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) s = fmaf(x[i][0], x[i][0], fmaf(x[i][1], x[i][1], s));
#pragma unroll
        for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m);
        s = 1.f / sqrtf(s / (float) D + a.eps);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (c[i][k] < D) x[i][k] = x[i][k] * s * w[c[i][k]];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (kind < 2 && lane + 64 * i < half_rot) {
            const float2_t cs = trig[lane + 64 * i];
            const float r0 = x[i][0], r1 = x[i][1];
            x[i][0] = r0 * cs[0] - r1 * cs[1];
            x[i][1] = r0 * cs[1] + r1 * cs[0];
        }
    if (kind != 0 && !place.has_page) return;
    const bool q_half = a.q_f16 != 0u, kv_half = a.kv_f16 != 0u;
    void *dst = (void *) ap_pick(kind, (uint64_t) a.q_out, (uint64_t) a.k_pages, (uint64_t) a.v_pages);
    const uint64_t to = (kind == 0 ? (uint64_t) t * nq + own : place.token * nk + own) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (c[i][k] < D) ap_store1(dst, to + c[i][k], kind == 0 ? q_half : kv_half, x[i][k]);
}

}  // namespace

#define AP_KERNEL(LPH)                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) moearc_qkv_append_l##LPH##_k(QkvAppendArgs a) { ap_body<LPH, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(256) moearc_qkv_append_l##LPH##x3_k(QkvAppendArgs a) { ap_body<LPH, 3>(a); }
AP_KERNEL(8)
AP_KERNEL(16)
AP_KERNEL(32)
extern "C" __global__ void __launch_bounds__(256) moearc_qkv_append_any_k(QkvAppendArgs a) { ap_any_body(a); }
