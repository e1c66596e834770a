// A key / value cache held in 8 bits (layout: tcq_kv8.h): rows into it, rows out of it, and grouped-query attention over it.
#include "tcq_kv8.h"

namespace {

constexpr int KT = 256;          // threads of every kernel here

struct KvAppend {
    const u16 *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;    // strides in elements
    const int *cu, *start;
    i8 *k8, *v8;
    float* scale;
    u16* tail;
    int rows, most, H, D, nblk, bf16, vec;
};

// A value as the cache holds it: NaN as 0, an infinity as the block's largest code; 8 bits have neither.
__device__ __forceinline__ float kv_finite(float v, float amax) { return __builtin_isnan(v) ? 0.f : fminf(fmaxf(v, -amax), amax); }
__device__ __forceinline__ float kv_mag(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.f;
}

// grid (2 x blocks a sequence may touch, H, B): one block of keys (even x) or values (odd) of one head. The rows of a block that is not
// full come from the tail (those before start) and from the call: the block is quantized again from its 16-bit rows, so that its
// codes depend on its rows alone and not on how they came. The keys' pieces are 16 dims of a token (one 16-byte code word), the values'
// 16 tokens of two dims (two code words), so that every store is 16 bytes in place and no transposition goes through LDS.
// The rows of the newest two blocks go to the tail. Where that overwrites the rows that the first block reads (a newest block of its
// parity), the first block's workgroup writes them, after its reads.
template <int D>
__global__ __launch_bounds__(KT) void k_kv8_append(KvAppend a) {
    constexpr int U = 4 * D >= KT ? 4 * D / KT : 1;           // pieces of 16 dims per thread (keys)
    constexpr int W = 2 * D >= KT ? 2 * D / KT : 1;           // pieces of 16 tokens x 2 dims (values)
    __shared__ float red[KT / 64];
    const int b = blockIdx.z, h = blockIdx.y, val = blockIdx.x & 1, tid = threadIdx.x;
    const int s = max(0, a.start[b]), c0 = a.cu ? max(0, a.cu[b]) : b * a.most;
    int m = a.cu ? a.cu[b + 1] - c0 : a.most;
    m = min(min(m, a.most), a.rows - c0);
    const int cap = a.nblk * KB, e = s < cap ? s + min(m, cap - s) : s;
    if (m <= 0 || e <= s) return;
    const int j0 = s / KB, j1 = (e - 1) / KB, blk = j0 + (blockIdx.x >> 1), p0 = blk * KB;
    if (blk > j1) return;
    const u16* in = val ? a.v : a.k;
    const int64_t tok = val ? a.v_tok : a.k_tok, hd = val ? a.v_head : a.k_head;
    const size_t bh = (size_t)b * a.H + h;
    u16* const slots = a.tail + (bh * 4 + val) * (KB * D);     // + 2 * (KB * D) for slot 1
    const bool bf = a.bf16;
    auto row = [&](int p) -> const u16* {                      // 16-bit row of position p (start of the block <= p < e)
        return p < s ? slots + (size_t)(blk & 1) * 2 * (KB * D) + (p % KB) * D : in + (c0 + (int64_t)(p - s)) * tok + h * hd;
    };
    const bool keep = blk >= j1 - 1 && (blk == j0 || ((blk - j0) & 1));
    u16* const slot = slots + (size_t)(blk & 1) * 2 * (KB * D);
    float amax = 0.f;
    if (!val) {
        uint4_t raw[U][2];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = tid + i * KT, key = (u & 15) + 16 * (u / D), d0 = (u >> 4) % (D / 16) * 16, p = p0 + key;
            raw[i][0] = raw[i][1] = uint4_t{0, 0, 0, 0};
            if (u < 4 * D && p < e) {
                const u16* r = row(p) + d0;
                if (p < s || a.vec) {
                    raw[i][0] = gptr((const uint4_t*)r)[0];
                    raw[i][1] = gptr((const uint4_t*)r)[1];
                } else {
#pragma unroll
                    for (int x = 0; x < 16; ++x) raw[i][x >> 3][(x >> 1) & 3] |= (u32)gptr(r)[x] << (16 * (x & 1));
                }
            }
        }
        float v[U][16];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                v[i][x] = kv_value((u16)(raw[i][x >> 3][(x >> 1) & 3] >> (16 * (x & 1))), bf);
                amax = fmaxf(amax, kv_mag(v[i][x]));
            }
        amax = block_max(amax, red);                           // ends with a barrier: every read of the tail is done
        const float sc = token_scale(amax);
        const QScale S = qscale(sc);
        if (tid == 0) a.scale[(bh * a.nblk + blk) * 2] = sc;
        i8* out = a.k8 + (bh * a.nblk + blk) * (size_t)(KB * D);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = tid + i * KT, key = (u & 15) + 16 * (u / D), d0 = (u >> 4) % (D / 16) * 16, p = p0 + key;
            if (u >= 4 * D) break;
            u32 w[4];
#pragma unroll
            for (int x = 0; x < 16; ++x) v[i][x] = kv_finite(v[i][x], amax);
            q8_words<4>(v[i], S, w);
            *gptr((uint4_t*)(out + (size_t)u * 16)) = uint4_t{w[0], w[1], w[2], w[3]};
            if (keep && p >= s && p < e) {
                gptr((uint4_t*)(slot + key * D + d0))[0] = raw[i][0];
                gptr((uint4_t*)(slot + key * D + d0))[1] = raw[i][1];
            }
        }
    } else {
        u32 raw[W][16];                                        // token 16 (x / 4) + 4 lg + x % 4, dims d0, d0 + 1
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int u = tid + i * KT, d0 = 2 * (u % (D / 2)), lg = u / (D / 2);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int p = p0 + 16 * (x >> 2) + 4 * lg + (x & 3);
                raw[i][x] = 0;
                if (u < 2 * D && p < e) {
                    const u16* r = row(p) + d0;
                    raw[i][x] = p < s || a.vec ? *gptr((const u32*)r) : (u32)gptr(r)[0] | ((u32)gptr(r)[1] << 16);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int x = 0; x < 16; ++x)
                amax = fmaxf(amax, fmaxf(kv_mag(kv_value((u16)raw[i][x], bf)), kv_mag(kv_value((u16)(raw[i][x] >> 16), bf))));
        amax = block_max(amax, red);
        const float sc = token_scale(amax);
        const QScale S = qscale(sc);
        if (tid == 0) a.scale[(bh * a.nblk + blk) * 2 + 1] = sc;
        i8* out = a.v8 + (bh * a.nblk + blk) * (size_t)(KB * D);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int u = tid + i * KT, d0 = 2 * (u % (D / 2)), lg = u / (D / 2);
            if (u >= 2 * D) break;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float v[16];
                u32 w[4];
#pragma unroll
                for (int x = 0; x < 16; ++x) v[x] = kv_finite(kv_value((u16)(raw[i][x] >> (16 * y)), bf), amax);
                q8_words<4>(v, S, w);
                const int d = d0 + y;
                *gptr((uint4_t*)(out + (size_t)((d / 16 * 4 + lg) * 16 + d % 16) * 16)) = uint4_t{w[0], w[1], w[2], w[3]};
            }
            if (keep)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int key = 16 * (x >> 2) + 4 * lg + (x & 3), p = p0 + key;
                    if (p >= s && p < e) *gptr((u32*)(slot + key * D + d0)) = raw[i][x];
                }
        }
    }
    if (blk != j0) return;
    // the newest block of this block's parity, past it: all of its rows are the call's
    const int jx = (j1 - j0) & 1 ? j1 - 1 : j1;
    if (jx < j0 + 2) return;
    const int last = min(KB, e - jx * KB);
    const u16* src = in + (c0 + (int64_t)(jx * KB - s)) * tok + h * hd;
    if (a.vec) {
        for (int u = tid; u < last * (D / 8); u += KT) {
            const int key = u / (D / 8), c = u % (D / 8);
            gptr((uint4_t*)(slot + key * D))[c] = gptr((const uint4_t*)(src + key * tok))[c];
        }
    } else {
        for (int u = tid; u < last * D; u += KT) gptr(slot)[u] = gptr(src + (u / D) * tok)[u % D];
    }
}

struct KvRead {
    const i8 *k8, *v8;
    const float* scale;
    const int *first, *lens;
    char *k, *v;
    int n, H, D, nblk, dt;
};

// grid (2 x blocks a window may touch, H, B): one block of keys (even x) or values; k, v (B, n, H, D), row i of sequence b is
// position first[b] + i, zeros from lens[b] on.
template <int D>
__global__ __launch_bounds__(KT) void k_kv8_read(KvRead a) {
    const int b = blockIdx.z, h = blockIdx.y, val = blockIdx.x & 1, tid = threadIdx.x;
    const int first = max(0, a.first[b]), end = min(max(0, a.lens[b]), a.nblk * KB), blk = first / KB + (int)(blockIdx.x >> 1);
    const int64_t p0 = (int64_t)blk * KB;
    if (p0 >= (int64_t)first + a.n) return;
    const bool there = blk < a.nblk;
    const size_t at = ((size_t)b * a.H + h) * a.nblk + (there ? blk : 0);
    const float sc = there ? a.scale[at * 2 + val] : 0.f;
    const i8* in = (val ? a.v8 : a.k8) + at * (size_t)(KB * D);
    char* out = val ? a.v : a.k;
    const int es = a.dt == TCQ_F32 ? 4 : 2;
    auto row = [&](int key) -> char* {                         // where token key of the block goes, or nowhere
        const int64_t i = p0 + key - first;
        return i < 0 || i >= a.n ? nullptr : out + (((size_t)b * a.n + i) * a.H + h) * D * es;
    };
    if (!val) {
        for (int u = tid; u < 4 * D; u += KT) {
            const int key = (u & 15) + 16 * (u / D), d0 = (u >> 4) % (D / 16) * 16;
            char* o = row(key);
            if (!o) continue;
            uint4_t w = {0, 0, 0, 0};
            if (p0 + key < end) w = *gptr((const uint4_t*)(in + (size_t)u * 16));
            float v[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = (float)(i8)(w[x >> 2] >> (8 * (x & 3))) * sc;
            if (p0 + key >= end)
#pragma unroll
                for (int x = 0; x < 16; ++x) v[x] = 0.f;
            uint4_t* q = (uint4_t*)(o + (size_t)d0 * es);
            if (a.dt == TCQ_F32) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    gptr(q)[x] = uint4_t{__float_as_uint(v[4 * x]), __float_as_uint(v[4 * x + 1]), __float_as_uint(v[4 * x + 2]), __float_as_uint(v[4 * x + 3])};
            } else {
                u32 r[8];
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    r[x] = a.dt == TCQ_BF16 ? bf16x2(v[2 * x], v[2 * x + 1]) : (u32)f32_to_f16(v[2 * x]) | ((u32)f32_to_f16(v[2 * x + 1]) << 16);
                gptr(q)[0] = uint4_t{r[0], r[1], r[2], r[3]};
                gptr(q)[1] = uint4_t{r[4], r[5], r[6], r[7]};
            }
        }
    } else {
        for (int u = tid; u < 2 * D; u += KT) {
            const int d0 = 2 * (u % (D / 2)), lg = u / (D / 2);
            const i8* f = in + (size_t)((d0 / 16 * 4 + lg) * 16 + d0 % 16) * 16;
            uint4_t w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (there) {
                w[0] = gptr((const uint4_t*)f)[0];
                w[1] = gptr((const uint4_t*)f)[1];
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int key = 16 * (x >> 2) + 4 * lg + (x & 3);
                char* o = row(key);
                if (!o) continue;
                const bool in_ = p0 + key < end;
                const float v0 = in_ ? (float)(i8)(w[0][x >> 2] >> (8 * (x & 3))) * sc : 0.f;
                const float v1 = in_ ? (float)(i8)(w[1][x >> 2] >> (8 * (x & 3))) * sc : 0.f;
                if (a.dt == TCQ_F32) *gptr((uint2_t*)(o + (size_t)d0 * 4)) = uint2_t{__float_as_uint(v0), __float_as_uint(v1)};
                else
                    *gptr((u32*)(o + (size_t)d0 * 2)) =
                        a.dt == TCQ_BF16 ? bf16x2(v0, v1) : (u32)f32_to_f16(v0) | ((u32)f32_to_f16(v1) << 16);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- attention
struct KvAttend {
    const u16* q;
    int64_t q_tok, q_head;                   // strides in elements
    const int *cu, *lens;
    const i8 *k8, *v8;
    const float* scale;
    float *part, *stat;                      // (rows, Hq, S, D) and (rows, Hq, S, 2), S > 1
    u16* o;                                  // (rows, Hq, D)
    float sl;                                // score scale * log2 e
    int rows, most, G, Hk, nblk, causal, bf16, S;
};

constexpr float QC = 32512.f;    // query digits: 127 * 256, the largest value whose rounded high digit stays within 127
constexpr float PC = 32639.f;    // probability digits: 127 * 256 + 127
constexpr float DIG = 12582912.f + 128.f;   // 1.5 * 2^23 + 128: adding it leaves the rounded integer plus 128 in the low bits

// four values as two words of INT8 digits: value = 256 hi + lo, lo in [-128, 127]. f: value + DIG
__device__ __forceinline__ void digits(float f0, float f1, float f2, float f3, u32& hi, u32& lo) {
    const u32 a = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x05010400u);   // bytes lo0 + 128, lo1 + 128, hi0, hi1
    const u32 b = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x05010400u);
    hi = __builtin_amdgcn_perm(b, a, 0x07060302u);
    lo = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
}
__device__ __forceinline__ int4_t mma_i8(uint4_t a, uint4_t b, int4_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4_t, a), __builtin_bit_cast(int4_t, b), c, 0, 0, 0);
}

// One wave's share: 16 query rows (token, head of the group) against every fourth block of its split. Everything in INT8 MFMAs:
//   S^T = K Q^T   A = 16 keys x 64 dims as stored, B = the query rows as two INT8 digits each (q = 2^E (256 hi + lo) / 32512, E the
//                 row's exponent: within 2^-16 of the row's largest value), exact int32 sums;
//   O^T = V^T P^T A = 16 dims x 64 keys as stored, B = the probabilities of the block as two digits of p / 2^m in 1 / 32639 (m the
//                 block's own maximum: a block whose probabilities are all small keeps its digits), exact int32 sums.
// So the cache's bytes are never converted: an FP16 product would spend two instructions on every pair of them. Maximum, sum and
// outputs are FP32; the scales of a block enter with its exponent's factor (keys) and when its outputs are added (values).
template <int D>
__global__ __launch_bounds__(KT, D == 256 ? 1 : 2) void k_kv8_attend(KvAttend a) {
    constexpr int KS = D / 64, DTL = D / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lg = lane >> 4;
    const int split = blockIdx.x % a.S, tile = blockIdx.x / a.S, h = blockIdx.y, b = blockIdx.z;
    const int c0 = a.cu ? max(0, a.cu[b]) : b * a.most, count = a.cu ? a.cu[b + 1] - c0 : a.most;
    const int m = min(min(count, a.most), a.rows - c0);              // rows computed here
    const int L = min(max(a.lens[b], 0), a.nblk * KB);
    const int nrows = m * a.G, row0 = 16 * tile;
    if (row0 >= nrows) return;                                       // uniform
    const int r = row0 + lr, t = r / a.G, hq = h * a.G + (r - t * a.G);
    const bool on = r < nrows;
    auto sees = [&](int tt) { return a.causal ? min(max(L - count + tt + 1, 0), L) : L; };
    const int vend = on ? sees(t) : 0, all = sees(row0 / a.G), kend = sees((min(row0 + 16, nrows) - 1) / a.G);
    const bool part_off = row0 + 16 > nrows;
    const int nb = (kend + KB - 1) / KB, step = 4 * a.S;
    const size_t bh = (size_t)b * a.Hk + h;
    const i8* kb = a.k8 + bh * a.nblk * (size_t)(KB * D);
    const i8* vb = a.v8 + bh * a.nblk * (size_t)(KB * D);
    const float* sb = a.scale + bh * a.nblk * 2;
    uint4_t K[4][KS], V[DTL];
    auto load_k = [&](int j) {
        const i8* p = kb + (size_t)j * (KB * D);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) K[kt][ks] = *gptr((const uint4_t*)(p + kt * (16 * D) + ks * 1024 + lane * 16));
    };
    auto load_v = [&](int j) {
        const i8* p = vb + (size_t)j * (KB * D);
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) V[dt] = *gptr((const uint4_t*)(p + dt * 1024 + lane * 16));
    };
    int j = split * 4 + wave;
    float sk = 0.f, sv = 0.f;
    if (j < nb) {
        load_k(j);
        load_v(j);
        sk = sb[2 * j];
        sv = sb[2 * j + 1];
    }
    // the query row's digits: this lane's dims 64 ks + 16 lg .. + 15
    uint4_t Qh[KS], Ql[KS];
    int E = 0;
    float qbad = 0.f;
    {
        float v[KS][16], mx = 0.f;
        const u16* qp = a.q + (c0 + (int64_t)(on ? t : 0)) * a.q_tok + (int64_t)(on ? hq : h * a.G) * a.q_head + 16 * lg;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint4_t w0 = gptr((const uint4_t*)(qp + 64 * ks))[0], w1 = gptr((const uint4_t*)(qp + 64 * ks))[1];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                v[ks][x] = kv_value((u16)((x < 8 ? w0 : w1)[(x >> 1) & 3] >> (16 * (x & 1))), a.bf16);
                mx = fmaxf(mx, fabsf(v[ks][x]));
                qbad = __builtin_fmaf(v[ks][x], 0.f, qbad);          // NaN once a value is not finite
            }
        }
        mx = fmaxf(mx, lane_xor(mx, 16, lane));
        mx = fmaxf(mx, lane_xor(mx, 32, lane));
        qbad += lane_xor(qbad, 16, lane);
        qbad += lane_xor(qbad, 32, lane);
        if (qbad != 0.f) mx = 1.f;                                   // the row's scores become NaN below
        E = mx > 0.f ? __builtin_amdgcn_frexp_expf(mx) : 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float f[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) f[y] = __builtin_fmaf(__builtin_amdgcn_ldexpf(v[ks][4 * x + y], -E), QC, DIG);
                u32 hi, lo;
                digits(f[0], f[1], f[2], f[3], hi, lo);
                Qh[ks][x] = hi;
                Ql[ks][x] = lo;
            }
    }
    const float qs = a.sl / QC + qbad;
    float4_t O[DTL];
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt) O[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    float mr = -__builtin_inff(), l = 0.f;
    for (; j < nb; j += step) {
        const bool more = j + step < nb;
        const float c = __builtin_amdgcn_ldexpf(qs * sk, E), svc = sv;
        float f[16];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            int4_t hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                hi = mma_i8(K[kt][ks], Qh[ks], hi);
                lo = mma_i8(K[kt][ks], Ql[ks], lo);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) f[4 * kt + e] = (float)((hi[e] << 8) + lo[e]);
        }
        if (more) {
            load_k(j + step);
            sk = sb[2 * (j + step)];
            sv = sb[2 * (j + step) + 1];
        }
        const bool edge = j * KB + KB > all || part_off;             // uniform: some key of the block is hidden from some row
        u32 vis = 0xffffu;
        if (edge) {
            vis = 0;
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (j * KB + 16 * (x >> 2) + 4 * lg + (x & 3) < vend) vis |= 1u << x;
#pragma unroll
            for (int x = 0; x < 16; ++x) f[x] = vis >> x & 1 ? f[x] : -__builtin_inff();
        }
        float mx = f[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) mx = fmaxf(mx, f[x]);
        mx = fmaxf(mx, lane_xor(mx, 16, lane));
        mx = fmaxf(mx, lane_xor(mx, 32, lane));
        const bool none = mx == -__builtin_inff();                   // the row sees no key of the block
        const float mb = none ? 0.f : mx * c;
        float p[16], lb = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(f[x], c, -mb));
        if (edge)
#pragma unroll
            for (int x = 0; x < 16; ++x) p[x] = vis >> x & 1 ? p[x] : 0.f;   // also where c is 0 and the product above NaN
#pragma unroll
        for (int x = 0; x < 16; ++x) lb += p[x];
        uint4_t Ph, Pl;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            u32 hi, lo;
            digits(__builtin_fmaf(p[4 * x], PC, DIG), __builtin_fmaf(p[4 * x + 1], PC, DIG), __builtin_fmaf(p[4 * x + 2], PC, DIG),
                   __builtin_fmaf(p[4 * x + 3], PC, DIG), hi, lo);
            Ph[x] = hi;
            Pl[x] = lo;
        }
        const float mn = none ? mr : fmaxf(mr, mb);
        if (__builtin_amdgcn_ballot_w64(mn > mr)) {                  // uniform: some row's maximum grew
            const float al = mn > mr ? __builtin_amdgcn_exp2f(mr - mn) : 1.f;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[dt][e] *= al;
            mr = mn;
        }
        const float w = none ? 0.f : __builtin_amdgcn_exp2f(mb - mr);
        l = __builtin_fmaf(w, lb, l);
        const float be = none ? 0.f : w * svc * (1.f / PC);
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) {
            const int4_t z = {0, 0, 0, 0};
            const int4_t hi = mma_i8(V[dt], Ph, z), lo = mma_i8(V[dt], Pl, z);
#pragma unroll
            for (int e = 0; e < 4; ++e) O[dt][e] = __builtin_fmaf((float)((hi[e] << 8) + lo[e]), be, O[dt][e]);
        }
        if (more) load_v(j + step);
    }
    // merge the four waves through LDS: statistics and outputs, wave w summing its quarter of the dims
    float4_t* x = (float4_t*)lds;
    float *sm = (float*)(lds + 4 * DTL * 1024), *sl = sm + 64;
    l += lane_xor(l, 16, lane);
    l += lane_xor(l, 32, lane);
    if (lg == 0) {
        sm[16 * wave + lr] = mr;
        sl[16 * wave + lr] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DTL; ++dt) x[(wave * DTL + dt) * 64 + lane] = O[dt];
    __syncthreads();
    float mx = -__builtin_inff(), lsum = 0.f, wt[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm[16 * w + lr]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        // a wave without a visible key has l = 0 and weight 0; one whose scores are NaN has l = NaN and weight NaN
        const float mw = sm[16 * w + lr], lw = sl[16 * w + lr];
        wt[w] = mw == -__builtin_inff() ? lw : __builtin_amdgcn_exp2f(mw - mx);
        lsum = __builtin_fmaf(wt[w], lw, lsum);
    }
    if (!on) return;
    const size_t row = (size_t)(c0 + t) * (a.Hk * a.G) + hq;
    if (a.S > 1 && wave == 0 && lg == 0) {
        a.stat[(row * a.S + split) * 2] = mx;
        a.stat[(row * a.S + split) * 2 + 1] = lsum;
    }
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;                // a row that sees no key: zeros
#pragma unroll
    for (int k = 0; k < DTL / 4; ++k) {
        const int dt = wave * (DTL / 4) + k;
        float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4_t v = x[(w * DTL + dt) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(wt[w], v[e], s[e]);
        }
        if (a.S > 1) {
            *gptr((float4_t*)(a.part + (row * a.S + split) * D + 16 * dt + 4 * lg)) = s;
        } else {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = s[e] * inv;
            const uint2_t u = a.bf16 ? uint2_t{bf16x2(f[0], f[1]), bf16x2(f[2], f[3])}
                                     : uint2_t{(u32)f32_to_f16(f[0]) | ((u32)f32_to_f16(f[1]) << 16), (u32)f32_to_f16(f[2]) | ((u32)f32_to_f16(f[3]) << 16)};
            *gptr((uint2_t*)(a.o + row * D + 16 * dt + 4 * lg)) = u;
        }
    }
}

// grid (most x Hq, 1, B): the splits' outputs of one row, weights exp2(m_s - max m), thread (g, 4 dims) summing every
// (KT / (D / 4))th split
template <int D>
__global__ __launch_bounds__(KT) void k_kv8_join(KvAttend a) {
    constexpr int TD = D / 4, NG = KT / TD;
    __shared__ float4_t sums[NG][TD];
    const int tid = threadIdx.x, d = tid % TD, g = tid / TD, S = a.S, b = blockIdx.z, Hq = a.Hk * a.G, t = blockIdx.x / Hq;
    const int c0 = a.cu ? max(0, a.cu[b]) : b * a.most;
    if (t >= min(a.cu ? a.cu[b + 1] - c0 : a.most, a.rows - c0)) return;
    const size_t row = (size_t)(c0 + t) * Hq + (blockIdx.x - t * Hq);
    const float* st = a.stat + row * S * 2;
    float mx = -__builtin_inff(), L = 0.f;
    for (int s = 0; s < S; ++s) mx = fmaxf(mx, st[2 * s]);
    for (int s = 0; s < S; ++s) L = __builtin_fmaf(st[2 * s] == -__builtin_inff() ? st[2 * s + 1] : __builtin_amdgcn_exp2f(st[2 * s] - mx), st[2 * s + 1], L);
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = g; s < S; s += NG) {
        const float w = st[2 * s] == -__builtin_inff() ? st[2 * s + 1] : __builtin_amdgcn_exp2f(st[2 * s] - mx);
        const float4_t v = *gptr((const float4_t*)(a.part + (row * S + s) * D + 4 * d));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(w, v[e], acc[e]);
    }
    sums[g][d] = acc;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int k = 1; k < NG; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += sums[k][d][e];
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    const uint2_t u = a.bf16 ? uint2_t{bf16x2(acc[0], acc[1]), bf16x2(acc[2], acc[3])}
                             : uint2_t{(u32)f32_to_f16(acc[0]) | ((u32)f32_to_f16(acc[1]) << 16), (u32)f32_to_f16(acc[2]) | ((u32)f32_to_f16(acc[3]) << 16)};
    *gptr((uint2_t*)(a.o + row * D + 4 * d)) = u;
}

bool kv_dim(int D) { return D == 64 || D == 128 || D == 256; }
bool kv_size(int B, int H, int nblk) { return B > 65535 || H > 65535 || nblk > (1 << 25) - 1; }

// Workgroups over which the blocks of a (sequence, KV head, 16 rows) are split: until the launch fills the chip, each wave keeping a block
int kv_splits(int B, int most, int G, int Hk, int keys) {
    const int64_t groups = (int64_t)B * Hk * (((int64_t)most * G + 15) / 16);
    const int nb = (keys + KB - 1) / KB;
    const int64_t want = (512 + groups - 1) / groups, can = (nb + 3) / 4;
    return (int)max((int64_t)1, min(min(want, can), (int64_t)256));
}

}  // namespace

#define KV_BY_DIM(CALL)              \
    do {                             \
        if (D == 256) CALL(256);     \
        else if (D == 128) CALL(128);\
        else CALL(64);               \
    } while (0)

extern "C" int tcq_kv8_append(const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, int dtype,
                              const int32_t* cu, const int32_t* start, int rows, int most, int B, int H, int D, int nblk, int8_t* k8,
                              int8_t* v8, float* scale, void* tail, tcq_stream_t stream) {
    if (!k || !v || !start || !k8 || !v8 || !scale || !tail || rows <= 0 || most <= 0 || B <= 0 || H <= 0 || nblk <= 0) return TCQ_ERR_ARG;
    if (dtype != TCQ_BF16 && dtype != TCQ_F16) return TCQ_ERR_DTYPE;
    if (!kv_dim(D) || kv_size(B, H, nblk)) return TCQ_ERR_UNSUPPORTED;
    if (!cu && (int64_t)most * B > rows) return TCQ_ERR_SHAPE;
    if (((uintptr_t)k | (uintptr_t)v) % 2 || ((uintptr_t)k8 | (uintptr_t)v8 | (uintptr_t)tail) % 16 || (uintptr_t)scale % 8) return TCQ_ERR_ALIGN;
    const int vec = !(((uintptr_t)k | (uintptr_t)v) % 16) && !((k_tok | k_head | v_tok | v_head) % 8);
    const KvAppend a = {(const u16*)k, (const u16*)v, k_tok, k_head, v_tok, v_head, cu, start, (i8*)k8, (i8*)v8, scale, (u16*)tail,
                        rows, most, H, D, nblk, dtype == TCQ_BF16, vec};
    const int64_t blocks = min((int64_t)nblk, ((int64_t)most + KB - 2) / KB + 1);
#define KV_APPEND(N) launch_k(k_kv8_append<N>, dim3((u32)(2 * blocks), H, B), dim3(KT), 0, (hipStream_t)stream, a)
    KV_BY_DIM(KV_APPEND);
#undef KV_APPEND
    return launch_status();
}

extern "C" int tcq_kv8_read(const int8_t* k8, const int8_t* v8, const float* scale, const int32_t* first, const int32_t* lens, int n, int B, int H,
                            int D, int nblk, void* k, void* v, int dtype, tcq_stream_t stream) {
    if (!k8 || !v8 || !scale || !first || !lens || !k || !v || n <= 0 || B <= 0 || H <= 0 || nblk <= 0) return TCQ_ERR_ARG;
    if (dtype != TCQ_BF16 && dtype != TCQ_F16 && dtype != TCQ_F32) return TCQ_ERR_DTYPE;
    if (!kv_dim(D) || kv_size(B, H, nblk)) return TCQ_ERR_UNSUPPORTED;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k8 | (uintptr_t)v8) % 16 || (uintptr_t)scale % 8) return TCQ_ERR_ALIGN;
    const KvRead a = {(const i8*)k8, (const i8*)v8, scale, first, lens, (char*)k, (char*)v, n, H, D, nblk, dtype};
    const int64_t blocks = ((int64_t)n + KB - 2) / KB + 1;
#define KV_READ(N) launch_k(k_kv8_read<N>, dim3((u32)(2 * blocks), H, B), dim3(KT), 0, (hipStream_t)stream, a)
    KV_BY_DIM(KV_READ);
#undef KV_READ
    return launch_status();
}

extern "C" int64_t tcq_kv8_attend_floats(int rows, int most, int B, int Hq, int Hk, int D, int keys) {
    if (rows <= 0 || most <= 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || keys < 0 || !kv_dim(D)) return 0;
    const int S = kv_splits(B, most, Hq / Hk, Hk, keys);
    return S > 1 ? (int64_t)rows * Hq * S * (D + 2) : 0;
}

extern "C" int tcq_kv8_attend(const void* q, int64_t q_tok, int64_t q_head, int dtype, const int32_t* cu, const int32_t* lens, int rows, int most,
                              int B, int Hq, int Hk, int D, int nblk, const int8_t* k8, const int8_t* v8, const float* scale, int causal,
                              float score_scale, int keys, float* part, void* o, tcq_stream_t stream) {
    if (!q || !lens || !k8 || !v8 || !scale || !o || rows <= 0 || most <= 0 || B <= 0 || Hq <= 0 || Hk <= 0 || nblk <= 0 || keys < 0 ||
        !(score_scale >= 0.f && score_scale < __builtin_inff()))
        return TCQ_ERR_ARG;
    if (dtype != TCQ_BF16 && dtype != TCQ_F16) return TCQ_ERR_DTYPE;
    if (Hq % Hk || (!cu && (int64_t)most * B > rows)) return TCQ_ERR_SHAPE;
    if (!kv_dim(D) || kv_size(B, Hk, nblk)) return TCQ_ERR_UNSUPPORTED;
    const int G = Hq / Hk, S = kv_splits(B, most, G, Hk, keys);
    const int64_t tiles = ((int64_t)most * G + 15) / 16;
    if (tiles * S > 0x7fffffff || (int64_t)most * Hq > 0x7fffffff || (int64_t)rows * Hq > 0x7fffffff) return TCQ_ERR_UNSUPPORTED;
    if (S > 1 && !part) return TCQ_ERR_ARG;
    if (((uintptr_t)q | (uintptr_t)k8 | (uintptr_t)v8 | (uintptr_t)o | (uintptr_t)part) % 16 || (q_tok | q_head) % 8 || (uintptr_t)scale % 8)
        return TCQ_ERR_ALIGN;
    KvAttend a = {(const u16*)q, q_tok, q_head, cu, lens, (const i8*)k8, (const i8*)v8, scale, part, part + (S > 1 ? (size_t)rows * Hq * S * D : 0),
                  (u16*)o, score_scale * 1.44269504088896341f, rows, most, G, Hk, nblk, causal != 0, dtype == TCQ_BF16, S};
    hipStream_t st = (hipStream_t)stream;
#define KV_ATTEND(N)                                                                                                    \
    do {                                                                                                                \
        launch_k(k_kv8_attend<N>, dim3((u32)(tiles * S), Hk, B), dim3(KT), (size_t)4 * (N / 16) * 1024 + 512, st, a);   \
        if (S > 1) {                                                                                                    \
            const int e = launch_status();                                                                              \
            if (e) return e;                                                                                            \
            launch_k(k_kv8_join<N>, dim3((u32)most * Hq, 1, B), dim3(KT), 0, st, a);                                          \
        }                                                                                                               \
    } while (0)
    KV_BY_DIM(KV_ATTEND);
#undef KV_ATTEND
    return launch_status();
}
