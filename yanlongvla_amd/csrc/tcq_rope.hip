// Rotary positions with several axes (time, height, width): pair i of a head turns by pos[axis[i]] * freq[i].
//
// The angle is taken in turns in FP64 (pos * freq / 2 pi, minus its nearest whole number) and only then rounded to FP32: at
// position 100000 an FP32 product is off by 4e-3 rad, this one by 1e-11 before the FP32 rounding of a number below one half (up to
// 9e-8 rad: for FP32 rows what it cuts off is put back in first order, 4.1e-8 relative against 64 bits instead of 5.9e-8). A workgroup
// computes the cosines and sines of its tokens once, into LDS, while the loads of its rows are in flight; every head of the token then
// uses them. MI355X: 4761 tokens of 32 heads x 64, FP32, 13.8 us (78 MB, 5.7 TB/s, some of it out of the last-level cache: memory
// bound), 2048 tokens of 24 heads x 128, BF16, 7.7 us (25 MB, 3.3 TB/s: launch, the FP64 angles and one wave of loads per workgroup),
// one token of the same 2.7 us.
#include "tcq_device.h"
#include "tcq_launch.h"

namespace {

constexpr int RT = 256;          // threads
constexpr int RTAB = 512;        // cosine / sine pairs of a workgroup's tokens in LDS
constexpr int RU = 4;            // pieces (of 16-byte halves) that a thread holds at a time

struct RopeHeads {
    const char* x;
    char* y;
    int64_t x_tok, x_head, y_tok, y_head;   // strides in bytes
    int heads;
};
struct RopeArgs {
    RopeHeads p[2];
    const void* pos;
    int64_t pos_axis, pos_tok;              // strides in elements
    const double* freq;
    const int* axis;
    int pos64, A, M, D, R, inverse;
};

template <int DT>
__device__ __forceinline__ float rope_get(const char* p) {
    return DT == TCQ_F32 ? *gptr((const float*)p) : DT == TCQ_BF16 ? bf16_to_f32(*gptr((const u16*)p)) : f16_to_f32(*gptr((const u16*)p));
}
template <int DT>
__device__ __forceinline__ void rope_put(char* p, float v) {
    if (DT == TCQ_F32) *gptr((float*)p) = v;
    else *gptr((u16*)p) = DT == TCQ_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}
// 16 bytes <-> the 4 (FP32) or 8 values they hold
template <int DT, int E>
__device__ __forceinline__ void rope_unpack(uint4_t w, float (&v)[E]) {
#pragma unroll
    for (int k = 0; k < E; ++k)
        v[k] = DT == TCQ_F32    ? __uint_as_float(w[k])
               : DT == TCQ_BF16 ? __uint_as_float((k & 1) ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16)
                                : f16_to_f32((u16)(w[k >> 1] >> (16 * (k & 1))));
}
template <int DT, int E>
__device__ __forceinline__ uint4_t rope_pack(const float (&v)[E]) {
    uint4_t w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = DT == TCQ_F32    ? __float_as_uint(v[k])
               : DT == TCQ_BF16 ? bf16x2(v[2 * k % E], v[(2 * k + 1) % E])
                                : (u32)f32_to_f16(v[2 * k % E]) | ((u32)f32_to_f16(v[(2 * k + 1) % E]) << 16);
    return w;
}

// cosine and sine of the pairs of tokens t0 .. t0 + n - 1 into cs (n x R / 2); an axis outside 0 .. A - 1 turns by nothing
template <int DT>
__device__ __forceinline__ void rope_table(const RopeArgs& a, int t0, int n, float2_t* cs) {
    const int half = a.R >> 1;
    for (int i = threadIdx.x; i < n * half; i += RT) {
        const int t = i / half, f = i - t * half, ax = a.axis ? gptr(a.axis)[f] : 0;
        double turns = 0.0;
        if (ax >= 0 && ax < a.A) {
            const int64_t at = ax * a.pos_axis + (t0 + t) * a.pos_tok;
            const double p = a.pos64 ? (double)gptr((const int64_t*)a.pos)[at] : (double)gptr((const int*)a.pos)[at];
            turns = p * gptr(a.freq)[f] * 0.15915494309189535;            // 1 / (2 pi)
            turns -= __builtin_rint(turns);
        }
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        if constexpr (DT == TCQ_F32) {
            const float e = (float)((turns - (double)(float)turns) * 6.283185307179586), c0 = c;
            c = __builtin_fmaf(-s, e, c);
            s = __builtin_fmaf(c0, e, s);
        }
        cs[i] = float2_t{c, a.inverse ? -s : s};
    }
}

// grid ceil(M / TT): the pieces (of E pairs) of a head on neighbouring threads, so a wave's loads are runs of whole rows; thread (g, c) takes
// piece c of the head rows (token, head) g, g + G, ... of the workgroup's TT tokens, whose token and head it steps by the quotient and
// remainder of G by the heads. ADJ: pairs are neighbours (2 i, 2 i + 1) and a piece is 16 bytes of E / 2 pairs; else they lie R / 2 apart
// and a piece is two times 16 bytes. The columns from R on are copied where the output is another tensor.
template <int DT, bool ADJ>
__global__ __launch_bounds__(RT) void k_rope(RopeArgs a, int TT) {
    constexpr int ES = DT == TCQ_F32 ? 4 : 2, E = 16 / ES, N = ADJ ? 1 : 2;
    __shared__ __attribute__((aligned(16))) float2_t cs[RTAB];
    const int half = a.R >> 1, t0 = blockIdx.x * TT, n = min(TT, a.M - t0), H = a.p[0].heads + a.p[1].heads;
    const int NP = ADJ ? a.R / E : half / E, G = RT / NP, c = threadIdx.x % NP, g = threadIdx.x / NP, dt = G / H, dh = G - dt * H;
    int t = g < G ? g / H : n, h = g - t * H;                             // (threads past the last whole group have no rows)
    const float2_t* tab = cs + (ADJ ? c * (E / 2) : c * E);
    uint4_t v[RU][N];
    char* out[RU];
    int tt[RU];
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            tt[i] = t;
            if (t < n) {
                const bool second = h >= a.p[0].heads;
                const RopeHeads& p = a.p[second];
                const int hh = second ? h - a.p[0].heads : h;
                const char* x = p.x + (t0 + t) * p.x_tok + hh * p.x_head + c * 16;
                out[i] = p.y + (t0 + t) * p.y_tok + hh * p.y_head + c * 16;
#pragma unroll
                for (int k = 0; k < N; ++k) v[i][k] = *gptr((const uint4_t*)(x + (size_t)(k * half * ES)));
            }
            t += dt;
            h += dh;
            if (h >= H) h -= H, ++t;
        }
    };
    load();
    rope_table<DT>(a, t0, n, cs);
    __syncthreads();
    for (;;) {
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            if (tt[i] >= n) break;
            const float2_t* w = tab + tt[i] * half;
            float p[E], q[E];
            rope_unpack<DT>(v[i][0], p);
            if constexpr (ADJ) {
#pragma unroll
                for (int k = 0; k < E; k += 2) {
                    const float lo = p[k], hi = p[k + 1];
                    p[k] = __builtin_fmaf(lo, w[k >> 1].x, -(hi * w[k >> 1].y));
                    p[k + 1] = __builtin_fmaf(hi, w[k >> 1].x, lo * w[k >> 1].y);
                }
            } else {
                rope_unpack<DT>(v[i][N - 1], q);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float lo = p[k], hi = q[k];
                    p[k] = __builtin_fmaf(lo, w[k].x, -(hi * w[k].y));
                    q[k] = __builtin_fmaf(hi, w[k].x, lo * w[k].y);
                }
                *gptr((uint4_t*)(out[i] + (size_t)(half * ES))) = rope_pack<DT>(q);
            }
            *gptr((uint4_t*)out[i]) = rope_pack<DT>(p);
        }
        if (t >= n) break;
        load();
    }
    const int NR = (a.D - a.R) / E, rest = n * H * NR;
    for (int u = threadIdx.x; u < rest; u += RT) {
        const int ut = u / (H * NR), w = u - ut * H * NR, uh = w / NR;
        const bool second = uh >= a.p[0].heads;
        const RopeHeads& p = a.p[second];
        const int hh = second ? uh - a.p[0].heads : uh;
        const int64_t at = (int64_t)a.R * ES + (int64_t)(w - uh * NR) * 16;
        const char* x = p.x + (t0 + ut) * p.x_tok + hh * p.x_head + at;
        char* y = p.y + (t0 + ut) * p.y_tok + hh * p.y_head + at;
        if (x != y) *gptr((uint4_t*)y) = *gptr((const uint4_t*)x);
    }
}

// Rows, strides or widths that are no whole 16-byte pieces: grid (M, pairs in tables of RTAB), one pair a thread.
template <int DT>
__global__ __launch_bounds__(RT) void k_rope_any(RopeArgs a, int adj) {
    constexpr int ES = DT == TCQ_F32 ? 4 : 2;
    const int t = blockIdx.x, half = a.R >> 1, H = a.p[0].heads + a.p[1].heads;
    __shared__ float2_t cs[RTAB];
    for (int f0 = 0; f0 < half; f0 += RTAB) {
        const int nf = min(RTAB, half - f0);
        RopeArgs part = a;
        part.R = 2 * nf;
        part.freq += f0;
        if (part.axis) part.axis += f0;
        __syncthreads();
        rope_table<DT>(part, t, 1, cs);
        __syncthreads();
        for (int u = threadIdx.x; u < H * nf; u += RT) {
            const int h = u / nf, f = u - h * nf;
            const bool second = h >= a.p[0].heads;
            const RopeHeads& p = a.p[second];
            const int hh = second ? h - a.p[0].heads : h;
            const int i = adj ? 2 * (f0 + f) : f0 + f, j = adj ? i + 1 : i + half;
            const char* x = p.x + t * p.x_tok + hh * p.x_head;
            char* y = p.y + t * p.y_tok + hh * p.y_head;
            const float lo = rope_get<DT>(x + (size_t)i * ES), hi = rope_get<DT>(x + (size_t)j * ES);
            const float2_t w = cs[f];
            rope_put<DT>(y + (size_t)i * ES, __builtin_fmaf(lo, w.x, -(hi * w.y)));
            rope_put<DT>(y + (size_t)j * ES, __builtin_fmaf(hi, w.x, lo * w.y));
        }
    }
    for (int u = threadIdx.x; u < H * (a.D - a.R); u += RT) {
        const int h = u / (a.D - a.R), c = a.R + u - h * (a.D - a.R);
        const bool second = h >= a.p[0].heads;
        const RopeHeads& p = a.p[second];
        const int hh = second ? h - a.p[0].heads : h;
        const char* x = p.x + t * p.x_tok + hh * p.x_head + (size_t)c * ES;
        char* y = p.y + t * p.y_tok + hh * p.y_head + (size_t)c * ES;
        if (x == y) continue;
        if (DT == TCQ_F32) *gptr((u32*)y) = *gptr((const u32*)x);
        else *gptr((u16*)y) = *gptr((const u16*)x);
    }
}

template <int DT>
void rope_launch(const RopeArgs& a, bool adj, bool vec, hipStream_t st) {
    if (!vec) {
        launch_k(k_rope_any<DT>, dim3(a.M), dim3(RT), 0, st, a, (int)adj);
        return;
    }
    // tokens a workgroup: about 1024 workgroups (2048 tokens of 24 heads x 128 BF16: 512 7.7 us, 1024 7.6, 2048 8.3; 4761 of 32 x 64 FP32 14.7 / 13.9 / 13.5)
    const int TT = max(1, min(RTAB / max(1, a.R >> 1), (a.M + 1023) / 1024));
    if (adj) launch_k(k_rope<DT, true>, dim3((a.M + TT - 1) / TT), dim3(RT), 0, st, a, TT);
    else launch_k(k_rope<DT, false>, dim3((a.M + TT - 1) / TT), dim3(RT), 0, st, a, TT);
}

}  // namespace

extern "C" int tcq_rope_axes(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head, int Hq,
                             const void* k, int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head, int Hk,
                             int dtype, const void* pos, int pos64, int64_t pos_axis, int64_t pos_tok, const double* freq,
                             const int32_t* axis, int A, int M, int D, int R, int adjacent, int inverse, tcq_stream_t stream) {
    if (!q || !q_out || Hq <= 0 || Hk < 0 || (Hk > 0 && (!k || !k_out)) || !pos || !freq || A <= 0 || M <= 0 || D <= 0) return TCQ_ERR_ARG;
    if (R <= 0 || R > D || R % 2) return TCQ_ERR_SHAPE;
    if (dtype != TCQ_F32 && dtype != TCQ_BF16 && dtype != TCQ_F16) return TCQ_ERR_DTYPE;
    const int es = dtype == TCQ_F32 ? 4 : 2, E = 16 / es;
    if (((uintptr_t)q | (uintptr_t)q_out | (Hk ? (uintptr_t)k | (uintptr_t)k_out : 0)) % es) return TCQ_ERR_ALIGN;
    if ((uintptr_t)pos % (pos64 ? 8 : 4) || (uintptr_t)freq % 8 || (uintptr_t)axis % 4) return TCQ_ERR_ALIGN;
    if ((int64_t)(Hq + Hk) * D > (1 << 24)) return TCQ_ERR_UNSUPPORTED;
    RopeArgs a = {};
    a.p[0] = {(const char*)q, (char*)q_out, q_tok * es, q_head * es, qo_tok * es, qo_head * es, Hq};
    a.p[1] = {(const char*)k, (char*)k_out, k_tok * es, k_head * es, ko_tok * es, ko_head * es, Hk};
    a.pos = pos;
    a.pos_axis = pos_axis;
    a.pos_tok = pos_tok;
    a.freq = freq;
    a.axis = axis;
    a.pos64 = pos64;
    a.A = A;
    a.M = M;
    a.D = D;
    a.R = R;
    a.inverse = inverse;
    bool vec = R / 2 <= RTAB && R / 2 / E <= RT && (D - R) % E == 0 && (adjacent ? R % E == 0 : R % (2 * E) == 0);
    for (int i = 0; i < (Hk ? 2 : 1); ++i) {
        const RopeHeads& p = a.p[i];
        vec = vec && !(((uintptr_t)p.x | (uintptr_t)p.y) % 16) && !((p.x_tok | p.x_head | p.y_tok | p.y_head) % 16);
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TCQ_F32) rope_launch<TCQ_F32>(a, adjacent, vec, st);
    else if (dtype == TCQ_BF16) rope_launch<TCQ_BF16>(a, adjacent, vec, st);
    else rope_launch<TCQ_F16>(a, adjacent, vec, st);
    return launch_status();
}
