// Residual addition, RMSNorm and INT8 rows in one pass: h = x + r (rounded to the stream's type, an output), n = (h / rms(h))
// (offset + w), scale = max|n| / 127, q = rint(n / scale).
//
// The codes do not need the norm: n / scale = 127 m / max|m| with m = h (offset + w), so the sum of squares and max|m| are
// reduced together, one barrier a row, and the norm only enters the scale. The row stays in registers between the reduction
// and the codes. Statistics in FP32. Memory bound from a few hundred rows on (7 bytes a value in 16-bit types), else latency.
// MI355X, BF16: 4000 rows of 4096 22.9 us (115 MB, 5.0 TB/s: the rate of a large copy), one row of 2048 2.7 us (a launch, two memory
// latencies and one barrier).
#include "tcq_device.h"
#include "tcq_launch.h"

namespace {

struct Norm8 {
    const void *x, *r, *w;
    void* h;
    i8* q;
    int* q4;
    float* scale;
    int64_t ldx, ldr, ldh;       // in elements
    float eps, offset;
    int M, K, ldq;
};

template <int DT>
__device__ __forceinline__ float n8_get(const void* p, size_t i) {
    return DT == TCQ_F32 ? gptr((const float*)p)[i] : DT == TCQ_BF16 ? bf16_to_f32(gptr((const u16*)p)[i]) : f16_to_f32(gptr((const u16*)p)[i]);
}
// 8 consecutive values at element i (16-byte aligned)
template <int DT>
__device__ __forceinline__ void n8_raw(const void* p, size_t i, uint4_t (&w)[DT == TCQ_F32 ? 2 : 1]) {
    w[0] = *gptr((const uint4_t*)((const char*)p + i * (DT == TCQ_F32 ? 4 : 2)));
    if constexpr (DT == TCQ_F32) w[1] = *gptr((const uint4_t*)((const char*)p + i * 4 + 16));
}
template <int DT>
__device__ __forceinline__ void n8_vals(const uint4_t (&w)[DT == TCQ_F32 ? 2 : 1], float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if constexpr (DT == TCQ_F32) v[k] = __uint_as_float(w[k >> 2][k & 3]);
        else if constexpr (DT == TCQ_BF16) v[k] = __uint_as_float((k & 1) ? w[0][k >> 1] & 0xffff0000u : w[0][k >> 1] << 16);
        else v[k] = f16_to_f32((u16)(w[0][k >> 1] >> (16 * (k & 1))));
    }
}
// h rounded to the stream's type: v becomes the rounded values, w their bits
template <int DT>
__device__ __forceinline__ void n8_round(float (&v)[8], uint4_t (&w)[DT == TCQ_F32 ? 2 : 1]) {
    if constexpr (DT == TCQ_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k >> 2][k & 3] = __float_as_uint(v[k]);
    } else {
        if constexpr (DT == TCQ_BF16) bf16_pack<4>(v, (u32*)&w[0]);
        else
#pragma unroll
            for (int k = 0; k < 4; ++k) w[0][k] = (u32)f32_to_f16(v[2 * k]) | ((u32)f32_to_f16(v[2 * k + 1]) << 16);
        n8_vals<DT>(w, v);
    }
}
// What a row's sums say: its scale and the divisor of its codes. A value that is not finite (bad: its product with zero is NaN)
// makes the scale NaN, so that the row's products show it; a row of zeros, or one whose sum of squares overflows (its norm is
// zero then), has scale 1 and codes 0.
__device__ __forceinline__ void n8_scales(float sum, float big, float bad, float eps, int K, float& scale, float& step) {
    const float rms = 1.f / __builtin_sqrtf(sum / (float)K + eps), s = big * rms / 127.f;
    const bool none = big == 0.f || !(s > 0.f);                           // (zeros without an eps: s is 0 / 0)
    scale = bad != 0.f || (big > 0.f && __builtin_isnan(s)) ? __builtin_nanf("") : none ? 1.f : s;
    step = none ? __builtin_inff() : big / 127.f;
}
// the two words of 8 codes of columns k .. k + 7
__device__ __forceinline__ void n8_store(const Norm8& a, int row, int k, const u32* w) {
    if (a.q) *gptr((u64*)(a.q + (size_t)row * a.K + k)) = (u64)w[0] | ((u64)w[1] << 32);
    if (a.q4 && a.ldq == TCQ_LDQ_TOKEN_BLOCKS) *gptr((u64*)((i8*)a.q4 + tb_offset(row, k, a.K))) = (u64)w[0] | ((u64)w[1] << 32);
    else if (a.q4) {
        gptr(a.q4)[(size_t)(k >> 2) * a.ldq + row] = (int)w[0];
        gptr(a.q4)[(size_t)((k >> 2) + 1) * a.ldq + row] = (int)w[1];
    }
}

// grid M, W waves: lane i of the workgroup holds the row's 8-value pieces i, i + T, ... (NV of them).
template <int DT, int NV>
__global__ __launch_bounds__(1024) void k_norm8(Norm8 a) {
    constexpr int NW = DT == TCQ_F32 ? 2 : 1;
    __shared__ float red[3][16];
    const int row = blockIdx.x, tid = threadIdx.x, T = blockDim.x, lane = tid & 63, wave = tid >> 6, P = a.K >> 3;
    uint4_t xr[NV][NW], rr[NV][NW], wr[NV][NW];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * T;
        if (p < P) {
            n8_raw<DT>(a.x, (size_t)row * a.ldx + 8 * p, xr[i]);
            if (a.r) n8_raw<DT>(a.r, (size_t)row * a.ldr + 8 * p, rr[i]);
            n8_raw<DT>(a.w, 8 * p, wr[i]);
        }
    }
    float m[NV][8], sum = 0.f, big = 0.f, bad = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * T;
        if (p < P) {
            float w[8];
            n8_vals<DT>(xr[i], m[i]);
            if (a.r) {
                n8_vals<DT>(rr[i], w);
#pragma unroll
                for (int k = 0; k < 8; ++k) m[i][k] = m[i][k] + w[k];
                n8_round<DT>(m[i], xr[i]);
            }
            if (a.h) {
                char* o = (char*)a.h + ((size_t)row * a.ldh + 8 * p) * (DT == TCQ_F32 ? 4 : 2);
#pragma unroll
                for (int k = 0; k < NW; ++k) gptr((uint4_t*)o)[k] = xr[i][k];
            }
            n8_vals<DT>(wr[i], w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                sum = __builtin_fmaf(m[i][k], m[i][k], sum);
                m[i][k] = m[i][k] * (a.offset + w[k]);
                big = fmaxf(big, fabsf(m[i][k]));
                bad = __builtin_fmaf(m[i][k], 0.f, bad);
            }
        }
    }
    sum = wave_sum(sum);
    big = wave_max(big);
    bad = wave_sum(bad);
    if (T > 64) {
        if (lane == 0) {
            red[0][wave] = sum;
            red[1][wave] = big;
            red[2][wave] = bad;
        }
        __syncthreads();
        sum = bad = big = 0.f;
        for (int i = 0; i < (T >> 6); ++i) {
            sum += red[0][i];
            big = fmaxf(big, red[1][i]);
            bad += red[2][i];
        }
    }
    float scale, step;
    n8_scales(sum, big, bad, a.eps, a.K, scale, step);
    if (tid == 0) a.scale[row] = scale;
    const QScale S = qscale(step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * T;
        if (p < P) {
            u32 w[2];
            q8_words<2>(m[i], S, w);
            n8_store(a, row, 8 * p, w);
        }
    }
}

// Widths that are no whole 8-value pieces, and rows that are not 16-byte aligned: grid M, 256 threads, the row read twice (the
// second time from its output, where it has one: the output may be one of the inputs).
template <int DT>
__global__ __launch_bounds__(256) void k_norm8_any(Norm8 a) {
    __shared__ float red[3][4];
    const int row = blockIdx.x, tid = threadIdx.x;
    auto value = [&](int k) {
        const float v = n8_get<DT>(a.x, (size_t)row * a.ldx + k);
        if (!a.r) return v;
        const float s = v + n8_get<DT>(a.r, (size_t)row * a.ldr + k);
        return DT == TCQ_F32 ? s : DT == TCQ_BF16 ? bf16_to_f32(f32_to_bf16(s)) : f16_to_f32(f32_to_f16(s));
    };
    float sum = 0.f, big = 0.f, bad = 0.f;
    for (int k = tid; k < a.K; k += 256) {
        const float h = value(k), m = h * (a.offset + n8_get<DT>(a.w, k));
        if (a.h) {
            const size_t at = (size_t)row * a.ldh + k;
            if (DT == TCQ_F32) gptr((float*)a.h)[at] = h;
            else gptr((u16*)a.h)[at] = DT == TCQ_BF16 ? f32_to_bf16(h) : f32_to_f16(h);
        }
        sum = __builtin_fmaf(h, h, sum);
        big = fmaxf(big, fabsf(m));
        bad = __builtin_fmaf(m, 0.f, bad);
    }
    sum = wave_sum(sum);
    big = wave_max(big);
    bad = wave_sum(bad);
    if ((tid & 63) == 0) {
        red[0][tid >> 6] = sum;
        red[1][tid >> 6] = big;
        red[2][tid >> 6] = bad;
    }
    __syncthreads();
    sum = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    big = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    bad = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    float scale, step;
    n8_scales(sum, big, bad, a.eps, a.K, scale, step);
    if (tid == 0) a.scale[row] = scale;
    const QScale S = qscale(step);
    for (int k = tid; k < a.K; k += 256) {
        const float h = a.h ? n8_get<DT>(a.h, (size_t)row * a.ldh + k) : value(k);
        const float m[4] = {h * (a.offset + n8_get<DT>(a.w, k)), 0.f, 0.f, 0.f};
        u32 w;
        q8_words<1>(m, S, &w);
        if (a.q) gptr(a.q)[(size_t)row * a.K + k] = (i8)w;
        if (a.q4 && a.ldq == TCQ_LDQ_TOKEN_BLOCKS) gptr((i8*)a.q4)[tb_offset(row, k, a.K)] = (i8)w;
        else if (a.q4) gptr((i8*)a.q4)[((size_t)(k >> 2) * a.ldq + row) * 4 + (k & 3)] = (i8)w;
    }
}

template <int DT>
void norm8_launch(const Norm8& a, bool vec, hipStream_t st) {
    if (!vec) {
        launch_k(k_norm8_any<DT>, dim3(a.M), dim3(256), 0, st, a);
        return;
    }
    const int P = a.K >> 3;
    // few rows: as many waves as the row has pieces for (latency); many: one wave takes up to 4 pieces a lane
    const int nv = a.M <= 512 ? 1 : P <= 64 ? 1 : P <= 128 ? 2 : 4;
    int T = (((P + nv - 1) / nv) + 63) & ~63, NV = nv;
    while (T > 1024) {
        NV *= 2;
        T = (((P + NV - 1) / NV) + 63) & ~63;
    }
    switch (NV) {
        case 1: launch_k(k_norm8<DT, 1>, dim3(a.M), dim3(T), 0, st, a); break;
        case 2: launch_k(k_norm8<DT, 2>, dim3(a.M), dim3(T), 0, st, a); break;
        default: launch_k(k_norm8<DT, 4>, dim3(a.M), dim3(T), 0, st, a); break;
    }
}

}  // namespace

extern "C" int tcq_add_norm_quantize(const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w, float eps, float offset, int dtype,
                                     void* xout, int64_t ldo, int8_t* q, int32_t* q4, int ldq, float* scale, int M, int K,
                                     tcq_stream_t stream) {
    if (!x || !w || !scale || (!q && !q4) || M <= 0 || K <= 0 || (q4 && ldq != TCQ_LDQ_TOKEN_BLOCKS && ldq < M)) return TCQ_ERR_ARG;
    if (dtype != TCQ_F32 && dtype != TCQ_BF16 && dtype != TCQ_F16) return TCQ_ERR_DTYPE;
    if (K > 2 * TCQ_MAX_WIDTH || (q4 && K % (ldq == TCQ_LDQ_TOKEN_BLOCKS ? 16 : 4))) return TCQ_ERR_SHAPE;
    const int es = dtype == TCQ_F32 ? 4 : 2;
    if (((uintptr_t)x | (uintptr_t)r | (uintptr_t)w | (uintptr_t)xout) % es || (uintptr_t)scale % 4) return TCQ_ERR_ALIGN;
    if (q4 && (uintptr_t)q4 % (ldq == TCQ_LDQ_TOKEN_BLOCKS ? 16 : 4)) return TCQ_ERR_ALIGN;
    const Norm8 a = {x, r, w, xout, (i8*)q, (int*)q4, scale, ldx, ldr, ldo, eps, offset, M, K, ldq};
    const bool vec = K % 8 == 0 && !(((uintptr_t)x | (uintptr_t)r | (uintptr_t)w | (uintptr_t)xout) % 16) && !((uintptr_t)q % 8) &&
                     !((ldx | (r ? ldr : 0) | (xout ? ldo : 0)) * es % 16);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TCQ_F32) norm8_launch<TCQ_F32>(a, vec, st);
    else if (dtype == TCQ_BF16) norm8_launch<TCQ_BF16>(a, vec, st);
    else norm8_launch<TCQ_F16>(a, vec, st);
    return launch_status();
}
