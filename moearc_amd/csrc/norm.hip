// The residual update and norm between two halves of a block, one pass over a row:
//   z = y, or y / sqrt(mean(y^2) + eps) * w_post      (a norm after the half that made y)
//   h += scale * gate * z
//   x = h / sqrt(mean(h^2) + eps) * w_pre             (the norm before the next half)
// Without y the plain RMSNorm of h; without x the residual update alone. Bound by HBM: a row is read
// once, its values stay in registers between the two sums of squares and the stores. A row takes 16, 64,
// 256 or 1024 threads (the host picks by its length), each NV vectors of VEC floats; sums are f32, per
// thread and then over the threads in a fixed order, so results repeat bit for bit. Measured: 2048 rows of
// 2880, y f32, x f16 (83 MB) 13.8 us, 65,536 rows of 128 (67 MB) 11.1 us, both partly out of the last-level
// cache; one row 3.8 us.
#include "common.h"

namespace {

template <int VEC>
struct NormVec {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ NormVec<VEC> norm_load(const void *p, uint64_t i, bool half) {
    NormVec<VEC> r;
    if constexpr (VEC == 4) {
        if (half) {
            const u32x2_t w = *(const u32x2_t *) ((const uint16_t *) p + i);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t pair = w[k];  // a copy: bit_cast of a vector's element takes element 0
                const half2_t h = __builtin_bit_cast(half2_t, pair);
                r.v[2 * k] = (float) h[0];
                r.v[2 * k + 1] = (float) h[1];
            }
        } else {
            const float4_t f = *(const float4_t *) ((const float *) p + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) r.v[k] = f[k];
        }
    } else {
        r.v[0] = half ? (float) ((const _Float16 *) p)[i] : ((const float *) p)[i];
    }
    return r;
}

template <int VEC>
__device__ __forceinline__ void norm_store(void *p, uint64_t i, bool half, const NormVec<VEC> &r) {
    if constexpr (VEC == 4) {
        if (half) {
            const half2_t a = {(_Float16) r.v[0], (_Float16) r.v[1]}, b = {(_Float16) r.v[2], (_Float16) r.v[3]};
            *(u32x2_t *) ((uint16_t *) p + i) = u32x2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
        } else {
            *(float4_t *) ((float *) p + i) = float4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
        }
    } else {
        if (half) ((_Float16 *) p)[i] = (_Float16) r.v[0];
        else ((float *) p)[i] = r.v[0];
    }
}

// The sum over a row's TPR threads, in every one of them. red: a float per wave of the work-group.
template <int TPR>
__device__ __forceinline__ float norm_sum(float s, float *red) {
    s += dpp<0xB1>(s);   // quad_perm [1,0,3,2]
    s += dpp<0x4E>(s);   // quad_perm [2,3,0,1]
    s += dpp<0x141>(s);  // row_half_mirror
    s += dpp<0x140>(s);  // row_mirror
    if constexpr (TPR >= 64) {
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
    }
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = s;
        __syncthreads();
        s = red[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) s += red[w];
    }
    return s;
}

template <int TPR, int NV, int VEC>
__device__ __forceinline__ void norm_body(const NormArgs &a) {
    constexpr int THREADS = TPR < 256 ? 256 : TPR, ROWS = THREADS / TPR;
    __shared__ float red[2][TPR > 64 ? TPR / 64 : 1];
    const uint32_t row = blockIdx.x * ROWS + threadIdx.x / TPR, t = threadIdx.x % TPR;
    if (row >= a.n_rows) return;  // whole rows of threads: with more than 64 threads a row is a work-group
    const uint64_t base = (uint64_t) row * a.n_cols;
    const bool yh = a.y_f16, xh = a.x_f16;
    NormVec<VEC> h[NV];
    auto at = [&](int i) { return VEC * ((uint32_t) i * TPR + t); };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (at(i) < a.n_cols) h[i] = norm_load<VEC>(a.h, base + at(i), false);
        else
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[i].v[k] = 0.f;
    }
    if (a.y) {
        NormVec<VEC> z[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (at(i) < a.n_cols) z[i] = norm_load<VEC>(a.y, base + at(i), yh);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) z[i].v[k] = 0.f;
        }
        if (a.w_post) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) s = fmaf(z[i].v[k], z[i].v[k], s);
            const float r = 1.f / sqrtf(norm_sum<TPR>(s, red[0]) / (float) a.n_cols + a.eps);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at(i) < a.n_cols) {
                    const NormVec<VEC> w = norm_load<VEC>(a.w_post, at(i), false);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) z[i].v[k] = z[i].v[k] * r * w.v[k];
                }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at(i) < a.n_cols) {
                if (a.gate) {
                    const NormVec<VEC> g = norm_load<VEC>(a.gate, (uint64_t) row * a.gate_stride + at(i), false);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) z[i].v[k] *= g.v[k];
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[i].v[k] = fmaf(a.scale, z[i].v[k], h[i].v[k]);
                norm_store<VEC>(a.h, base + at(i), false, h[i]);
            }
    }
    if (!a.x) return;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s = fmaf(h[i].v[k], h[i].v[k], s);
    const float r = 1.f / sqrtf(norm_sum<TPR>(s, red[1]) / (float) a.n_cols + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at(i) < a.n_cols) {
            NormVec<VEC> o;
#pragma unroll
            for (int k = 0; k < VEC; ++k) o.v[k] = h[i].v[k] * r;
            if (a.w_pre) {
                const NormVec<VEC> w = norm_load<VEC>(a.w_pre, at(i), false);
#pragma unroll
                for (int k = 0; k < VEC; ++k) o.v[k] *= w.v[k];
            }
            norm_store<VEC>(a.x, base + at(i), xh, o);
        }
}

// Rows longer than the threads' registers hold: each pass reads the row again.
__device__ __forceinline__ void norm_long_body(const NormArgs &a) {
    __shared__ float red[2][16];
    const uint64_t base = (uint64_t) blockIdx.x * a.n_cols;
    const uint32_t t = threadIdx.x;
    float s = 0.f;
    if (a.y) {
        float r = 1.f;
        if (a.w_post) {
            for (uint32_t c = t; c < a.n_cols; c += 1024u) {
                const float v = norm_load<1>(a.y, base + c, a.y_f16).v[0];
                s = fmaf(v, v, s);
            }
            r = 1.f / sqrtf(norm_sum<1024>(s, red[0]) / (float) a.n_cols + a.eps);
        }
        s = 0.f;
        for (uint32_t c = t; c < a.n_cols; c += 1024u) {
            float z = norm_load<1>(a.y, base + c, a.y_f16).v[0];
            if (a.w_post) z = z * r * a.w_post[c];
            if (a.gate) z *= a.gate[(uint64_t) blockIdx.x * a.gate_stride + c];
            const float h = fmaf(a.scale, z, a.h[base + c]);
            a.h[base + c] = h;
            s = fmaf(h, h, s);
        }
    } else {
        for (uint32_t c = t; c < a.n_cols; c += 1024u) s = fmaf(a.h[base + c], a.h[base + c], s);
    }
    if (!a.x) return;
    const float r = 1.f / sqrtf(norm_sum<1024>(s, red[1]) / (float) a.n_cols + a.eps);
    for (uint32_t c = t; c < a.n_cols; c += 1024u) {  // each thread reads the h that it wrote
        const float o = a.h[base + c] * r;
        norm_store<1>(a.x, base + c, a.x_f16, NormVec<1>{{a.w_pre ? o * a.w_pre[c] : o}});
    }
}

}  // namespace

#define NORM_KERNEL(TPR, NV)                                                                                 \
    extern "C" __global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) moearc_norm_r##TPR##_v4_k(NormArgs a) { \
        norm_body<TPR, NV, 4>(a);                                                                            \
    }                                                                                                        \
    extern "C" __global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) moearc_norm_r##TPR##_v1_k(NormArgs a) { \
        norm_body<TPR, 4 * NV, 1>(a);                                                                        \
    }
NORM_KERNEL(16, 4)
NORM_KERNEL(64, 4)
NORM_KERNEL(256, 4)
NORM_KERNEL(1024, 4)
extern "C" __global__ void __launch_bounds__(1024) moearc_norm_long_k(NormArgs a) { norm_long_body(a); }
