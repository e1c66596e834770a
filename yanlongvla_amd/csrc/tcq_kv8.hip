// A key / value cache held in 8 bits (layout: tcq_kv8.h): rows into it, rows out of it, and grouped-query attention over it.
#include <type_traits>

#include "tcq_kv8.h"

namespace {

constexpr int KT = 256;          // threads
constexpr int MAX_SPLITS = 256;  // parts of one row's keys

struct KvAppend {
    const u16 *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;    // strides in elements
    const int *cu, *start;
    i8 *k8, *v8;
    float* scale;
    u16* tail;
    int rows, most, H, D, nblk, near;
};

// A value as the cache holds it: NaN as 0, an infinity as the block's largest code; 8 bits have neither.
__device__ __forceinline__ float kv_finite(float v, float amax) { return __builtin_isnan(v) ? 0.f : fminf(fmaxf(v, -amax), amax); }
__device__ __forceinline__ float kv_mag(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.f;
}

// grid (2 x blocks a sequence may touch, H, B), 4 D threads: one block of keys (even x) or values (odd) of one head, 16 values a thread. The
// rows of a block that is not full come from the tail (those before start) and from the call: the block is quantized again from its 16-bit
// rows, so that its codes depend on its rows alone and not on how they came. A thread holds 16 dims of a token (keys) or 16 tokens of a
// dim (values), which are the 16 bytes of one store, so no transposition goes through LDS. The largest magnitude is taken from the
// bits of two values at a time; only a block where that is no finite number looks at each value.
// The rows of the newest two blocks go to the tail. Where that overwrites the rows that the first block reads (a newest block of its
// parity), the first block's workgroup writes them, after its reads.
// MI355X: 4500 rows of 6 prompts, 8 heads of 128 11.5 us (28 MB: 2.4 TB/s; instruction issue, 14 us before whole blocks had one base address and
// 36 with 32 values a thread, a load waiting for each row's branch); one row each of 16 sequences, one head of 256, 7.2 us (latency).
template <int D, bool BF, bool VEC>
__global__ __launch_bounds__(4 * D) void k_kv8_append(KvAppend a) {
    __shared__ float red[16];
    const int b = blockIdx.z, h = blockIdx.y, val = blockIdx.x & 1, tid = threadIdx.x;
    const int s = max(0, a.start[b]), c0 = a.cu ? max(0, a.cu[b]) : b * a.most;
    const int m = min(min(a.cu ? a.cu[b + 1] - c0 : a.most, a.most), a.rows - c0);
    const int cap = a.nblk * KB, e = s < cap ? s + min(m, cap - s) : s;
    if (m <= 0 || e <= s) return;
    const int j0 = s / KB, j1 = (e - 1) / KB, blk = j0 + (blockIdx.x >> 1), p0 = blk * KB;
    if (blk > j1) return;
    const u16* in = val ? a.v : a.k;
    const int64_t tok = val ? a.v_tok : a.k_tok;
    in += h * (val ? a.v_head : a.k_head) + (c0 - (int64_t)s) * tok;               // row p of the sequence at in + p tok, for p >= s
    const size_t bh = (size_t)b * a.H + h;
    u16* const slots = a.tail + (bh * 4 + val) * (KB * D);     // + 2 * (KB * D) for slot 1
    u16* const slot = slots + (size_t)(blk & 1) * 2 * (KB * D);
    const bool keep = blk >= j1 - 1 && (blk == j0 || ((blk - j0) & 1));
    u32 raw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    // keys: dims d .. d + 15 of token t; values: tokens 16 (x / 4) + t + x % 4 of dim d, t = 4 lane group
    const int t = val ? tid / D * 4 : (tid & 15) + 16 * (tid / D), d = val ? tid % D : (tid >> 4) % (D / 16) * 16;
    u16 x[16];
    if (p0 >= s && p0 + KB <= e && a.near) {                   // uniform: a whole block of the call's rows, one base and 32-bit offsets
        const u16* base = in + (int64_t)p0 * tok;
        const u32 off = (u32)t * (u32)tok + (u32)d;
        if (val) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = gptr(base + (int64_t)(16 * (i >> 2) + (i & 3)) * tok)[off];
        } else if (VEC) {
            const uint4_t y = gptr((const uint4_t*)(base + off))[0], z = gptr((const uint4_t*)(base + off))[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = y[i], raw[4 + i] = z[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = gptr(base + off)[i];
        }
        if (val || !VEC)
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = (u32)x[2 * i] | ((u32)x[2 * i + 1] << 16);
    } else if (!val) {
        // (a row past the last one reads that one, so that no load waits for a branch, and counts as zeros)
        const int p = p0 + t;
        const u16* r = (p < s ? slot + t * D : in + (int64_t)min(p, e - 1) * tok) + d;
        if (VEC) {
            const uint4_t y = gptr((const uint4_t*)r)[0], z = gptr((const uint4_t*)r)[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = y[i], raw[4 + i] = z[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i >> 1] |= (u32)gptr(r)[i] << (16 * (i & 1));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = p < e ? raw[i] : 0;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = 16 * (i >> 2) + t + (i & 3), p = p0 + key;
            x[i] = gptr(p < s ? slot + key * D : in + (int64_t)min(p, e - 1) * tok)[d];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i >> 1] |= (u32)(p0 + 16 * (i >> 2) + t + (i & 3) < e ? x[i] : 0) << (16 * (i & 1));
    }
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, raw[i] & 0x7fff7fffu));
    const u16 bits = (u16)block_max((float)max(top.x, top.y), red);                 // ends with a barrier: every read of the tail is done
    float v[16], amax = kv_value(bits, BF);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = kv_value((u16)(raw[i >> 1] >> (16 * (i & 1))), BF);
    if (bits >= (BF ? 0x7f80 : 0x7c00)) {                                           // uniform
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, kv_mag(v[i]));
        amax = block_max(amax, red);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = kv_finite(v[i], amax);
    }
    const float sc = token_scale(amax);
    u32 w[4];
    // the code is rint(127 x / amax), both sides by 128: a 16-bit value times 127 is exact, so a value of half the largest is the tie that it is
    // (over the rounded scale it would fall to either side)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= 127.f / 128.f;
    q8_words<4>(v, qscale(amax > 0.f ? amax * 0x1p-7f : 1.f), w);
    const size_t at = bh * a.nblk + blk;
    if (tid == 0) a.scale[at * 2 + val] = sc;
    const int unit = val ? (d / 16 * 4 + t / 4) * 16 + d % 16 : tid;
    *gptr((uint4_t*)((val ? a.v8 : a.k8) + at * (KB * D) + (size_t)unit * 16)) = uint4_t{w[0], w[1], w[2], w[3]};
    if (keep) {
        if (!val) {
            if (p0 + t >= s && p0 + t < e) {
                gptr((uint4_t*)(slot + t * D + d))[0] = uint4_t{raw[0], raw[1], raw[2], raw[3]};
                gptr((uint4_t*)(slot + t * D + d))[1] = uint4_t{raw[4], raw[5], raw[6], raw[7]};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = 16 * (i >> 2) + t + (i & 3);
                if (p0 + key >= s && p0 + key < e) gptr(slot)[key * D + d] = (u16)(raw[i >> 1] >> (16 * (i & 1)));
            }
        }
    }
    if (blk != j0) return;
    // the newest block of this block's parity, past it: all of its rows are the call's
    const int jx = (j1 - j0) & 1 ? j1 - 1 : j1;
    if (jx < j0 + 2) return;
    const int last = min(KB, e - jx * KB);
    for (int u = tid; u < last * (D / 8); u += 4 * D) {
        const int key = u / (D / 8), c = u % (D / 8) * 8;
        const u16* r = in + (int64_t)(jx * KB + key) * tok + c;
        if (VEC) *gptr((uint4_t*)(slot + key * D + c)) = *gptr((const uint4_t*)r);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) gptr(slot)[key * D + c + i] = gptr(r)[i];
    }
}

struct KvRead {
    const i8 *k8, *v8;
    const float* scale;
    const int *first, *lens;
    char *k, *v;
    int n, H, D, nblk, dt;
};

__device__ __forceinline__ u32 kv_pair(float x, float y, int dt) {   // (finite values)
    return dt == TCQ_BF16 ? bf16_cvt2(x, y) : (u32)f32_to_f16(x) | ((u32)f32_to_f16(y) << 16);
}

// grid (2 x D / 64 x blocks a window may touch, H, B): 256 pieces of 16 values of a block's keys (even block index) or values; k, v (B, n, H, D),
// row i of sequence b is position first[b] + i, zeros from lens[b] on. MI355X: 6 x 1024 rows, 8 heads of 128 11.2 us (38 MB, 3.4 TB/s).
template <int D>
__global__ __launch_bounds__(KT) void k_kv8_read(KvRead a) {
    const int b = blockIdx.z, h = blockIdx.y, bx = blockIdx.x / (D / 64), val = bx & 1, u = blockIdx.x % (D / 64) * KT + threadIdx.x;
    const int first = max(0, a.first[b]), end = min(max(0, a.lens[b]), a.nblk * KB), blk = first / KB + (bx >> 1);
    const int64_t p0 = (int64_t)blk * KB;
    if (p0 >= (int64_t)first + a.n) return;
    const bool there = blk < a.nblk;
    const size_t at = ((size_t)b * a.H + h) * a.nblk + (there ? blk : 0);
    const int es = a.dt == TCQ_F32 ? 4 : 2;
    const int lo = (int)max((int64_t)0, first - p0), hi = (int)min((int64_t)KB, first + (int64_t)a.n - p0);   // tokens of the block in the window,
    const int have = (int)max((int64_t)0, min((int64_t)KB, end - p0));                                       // and those that it holds
    const size_t row = (size_t)a.H * D * es;                                         // bytes from row to row
    char* const out = (val ? a.v : a.k) + ((int64_t)b * a.n + (p0 - first)) * (int64_t)row + (size_t)h * D * es;
    const float sc = there ? a.scale[at * 2 + val] : 0.f;
    const i8* in = (val ? a.v8 : a.k8) + at * (size_t)(KB * D);
    if (!val) {
        const int key = (u & 15) + 16 * (u / D), d = (u >> 4) % (D / 16) * 16;
        if (key < lo || key >= hi) return;
        uint4_t w = {0, 0, 0, 0};
        if (key < have) w = *gptr((const uint4_t*)(in + (size_t)u * 16));
        float v[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) v[x] = i8_f32(w[x >> 2], x & 3) * sc;
        if (key >= have)                                                             // (a block that nothing was written to has any scale)
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = 0.f;
        uint4_t* q = (uint4_t*)(out + key * row + (size_t)d * es);
        if (a.dt == TCQ_F32) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                gptr(q)[x] = uint4_t{__float_as_uint(v[4 * x]), __float_as_uint(v[4 * x + 1]), __float_as_uint(v[4 * x + 2]), __float_as_uint(v[4 * x + 3])};
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
                gptr(q)[x] = uint4_t{kv_pair(v[8 * x], v[8 * x + 1], a.dt), kv_pair(v[8 * x + 2], v[8 * x + 3], a.dt),
                                     kv_pair(v[8 * x + 4], v[8 * x + 5], a.dt), kv_pair(v[8 * x + 6], v[8 * x + 7], a.dt)};
        }
    } else {
        const int d = 2 * (u % (D / 2)), lg = u / (D / 2) & 3, hf = u / (2 * D);     // tokens 32 hf + 16 (x / 4) + 4 lg + x % 4 of two dims
        const i8* f = in + (size_t)((d / 16 * 4 + lg) * 16 + d % 16) * 16 + 8 * hf;
        const uint2_t w0 = *gptr((const uint2_t*)f), w1 = *gptr((const uint2_t*)(f + 16));   // (of block 0 where there is none)
        const int t0 = 32 * hf + 4 * lg;
        char* q = out + t0 * row + (size_t)d * es;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const int key = t0 + 16 * (x >> 2) + (x & 3);
            if (key < lo || key >= hi) continue;
            const float v0 = key < have ? i8_f32(w0[x >> 2], x & 3) * sc : 0.f, v1 = key < have ? i8_f32(w1[x >> 2], x & 3) * sc : 0.f;
            char* o = q + (16 * (x >> 2) + (x & 3)) * row;
            if (a.dt == TCQ_F32) *gptr((uint2_t*)o) = uint2_t{__float_as_uint(v0), __float_as_uint(v1)};
            else *gptr((u32*)o) = kv_pair(v0, v1, a.dt);
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
    int last;                                // the row tile of blockIdx.z = 0
};

constexpr float QC = 32512.f;    // query digits: 127 * 256, the largest value whose rounded high digit stays within 127
constexpr float PC = 32639.f;    // probability digits: 127 * 256 + 127
constexpr int UP = 7;            // FP16 probabilities are raised by 2^7: up to 2^8 before the outputs are rescaled, so up to 2^15 of FP16's 2^16
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

__device__ __forceinline__ void store4(u16* o, float4_t v, bool bf16) {
    const uint2_t u = bf16 ? uint2_t{bf16x2(v[0], v[1]), bf16x2(v[2], v[3])}
                           : uint2_t{(u32)f32_to_f16(v[0]) | ((u32)f32_to_f16(v[1]) << 16), (u32)f32_to_f16(v[2]) | ((u32)f32_to_f16(v[3]) << 16)};
    *gptr((uint2_t*)o) = u;
}

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
// 16 codes -> two fragments' 8 FP16 values of a lane, exact
__device__ __forceinline__ void widen(uint4_t w, half8_t& a, half8_t& b) {
    uint4_t o[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const u32 u = w[k] ^ 0x80808080u;
        const half2_t off = {(_Float16)1152.f, (_Float16)1152.f};
        const half2_t x = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
        const half2_t y = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
        o[k >> 1][2 * (k & 1)] = __builtin_bit_cast(u32, x);
        o[k >> 1][2 * (k & 1) + 1] = __builtin_bit_cast(u32, y);
    }
    a = __builtin_bit_cast(half8_t, o[0]);
    b = __builtin_bit_cast(half8_t, o[1]);
}

// 16 RT query rows (token, head of the group) of one KV head, W waves that take its blocks in turn. The cache's bytes go from memory straight
// into MFMA fragments:
//   S^T = K Q^T   INT8, A = 16 keys x 64 dims as stored, B = the query rows as two digits each (q = 2^E (256 hi + lo) / 32512, E the
//                 row's exponent: within 2^-16 of the row's largest value), exact int32 sums, so the keys are never converted;
//   O^T = V^T P^T RT = 1: INT8, A = 16 dims x 64 keys as stored, B = the probabilities of the block as two digits of p / 2^m in 1 / 32639
//                 (m the block's own maximum: a block whose probabilities are all small keeps its digits), exact int32 sums that are
//                 scaled and added in FP32: nothing is converted, but every output is touched once a block.
//                 RT > 1: FP16, A = 16 dims x 32 keys widened in registers (two instructions for two values, for all RT tiles: the byte as
//                 the low half of 1024 + 128 + code, less 1152, exact), B = the probabilities times the block's value scale / 2^u, FP32
//                 sums that stay in the accumulators in units of 2^u, which every row has of its own, 2^-7 of a block's scale (the scale
//                 rides on the exponent; a unit that changes rescales the row's sums exactly); the probabilities' sum is their product
//                 with ones. Where the scales of a row's blocks lie so far apart that no unit holds both its sums and the block, the sum
//                 takes the probabilities all the same and the values' products are left at what FP16 has of them.
// The outputs are rescaled only once a maximum is a factor of 256 past the one that they stand on.
// A wave holds one block's keys or values at a time and leaves the overlap of loads, matrix and vector instructions to the other waves of
// its SIMD (four of them for D up to 128): one wave issues a vector instruction every 7 to 13 cycles here, four together every 3 to 5. With
// the next block's keys and values already under way (twice the registers, half the waves) 968 causal rows of 16 x 128 took 19.5 us instead
// of 16.6, 4096 rows 140 instead of 131 (both before the grid below). D = 256 in four waves, where two a SIMD are all that fit, does fetch
// the next keys: 131000 keys of two sequences 25.3 us instead of 27.5 (4.6 TB/s; 16 sequences of 8 heads x 128 behind 4 to 8 thousand keys
// 40.3 us, 5.1 TB/s).
// Range: scores of up to 2^26 (FP32 tells those past 2^23 apart by whole numbers only). RT = 1 holds the outputs in FP32 as they are, so values
// from about 1e-35 to 1e35 keep their digits; RT > 1 in units of the row's own.
// Grid (Hk x parts, B, row tiles): workgroups go to the eight XCDs in turn, so with eight KV heads an XCD's L2 sees one head's keys, and a
// tile's workgroups of all sequences come before the next tile's, the last tiles first, as they see the most keys. With the tiles of a head
// side by side and the first ones first: 968 causal rows of 16 x 128 15.3 us against 11.7, of 8 x 256 15.3 against 12.9, 4096 rows 117
// against 96, 90 rows behind 1846 keys, 8 sequences of 16 x 64 31.3 against 16.7 (2 x 1024 rows behind up to 4096 keys 92.6 against 93.4).
template <int D, int W, int RT>
__global__ __launch_bounds__(W * 64, D == 256 || RT == 2 ? 2 : 4) void k_kv8_attend(KvAttend a) {
    constexpr int KS = D / 64, DTL = D / 16;
    constexpr int QN = RT * KS;                                      // (tile, K step) pairs of query digits, one a wave
    static_assert(QN <= W, "a wave makes the digits of at most one pair");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lg = lane >> 4;
    const int split = blockIdx.x % a.S, h = blockIdx.x / a.S, b = blockIdx.y, tile = a.last - blockIdx.z;
    const int c0 = a.cu ? max(0, a.cu[b]) : b * a.most, count = a.cu ? a.cu[b + 1] - c0 : a.most;
    const int m = min(min(count, a.most), a.rows - c0);              // rows computed here
    const int n = max(a.lens[b], 0), L = min(n, a.nblk * KB);        // the length, which may go past the capacity, and what is held of it
    const int nrows = m * a.G, row0 = 16 * RT * tile;
    if (row0 >= nrows) return;                                       // uniform
    auto sees = [&](int tt) { return a.causal ? min(max(n - count + tt + 1, 0), L) : L; };
    auto token = [&](int r, int& hq) {                               // row r of the KV head: its token and query head
        const int t = r / a.G;
        hq = h * a.G + (r - t * a.G);
        return t;
    };
    const int all = __builtin_amdgcn_readfirstlane(sees(row0 / a.G));
    const int kend = __builtin_amdgcn_readfirstlane(sees((min(row0 + 16 * RT, nrows) - 1) / a.G));
    const int nb = (kend + KB - 1) / KB, step = W * a.S;
    const size_t bh = (size_t)b * a.Hk + h;
    const i8* kb = a.k8 + bh * a.nblk * (size_t)(KB * D);
    const i8* vb = a.v8 + bh * a.nblk * (size_t)(KB * D);
    const float* sb = a.scale + bh * a.nblk * 2;
    uint4_t K[4][KS], V[DTL];
    float sk = 0.f, sv = 0.f;
    auto load_k = [&](int j) {
        const i8* p = kb + (size_t)j * (KB * D);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) K[kt][ks] = *gptr((const uint4_t*)(p + kt * (16 * D) + ks * 1024 + lane * 16));
        sk = sb[2 * j];
        sv = sb[2 * j + 1];
    };
    auto load_v = [&](int j) {
        const i8* p = vb + (size_t)j * (KB * D);
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) V[dt] = *gptr((const uint4_t*)(p + dt * 1024 + lane * 16));
    };
    int j = split * W + wave;
    // the query rows' digits: wave KS rt + ks makes K step ks of tile rt, this lane's dims 64 ks + 16 lg .. + 15 of row lr, after the
    // maxima have met in LDS
    uint4_t wq[2];
    const int qt = wave / KS;
    if (wave < QN) {
        const int r = row0 + 16 * qt + lr;
        int hq;
        const int t = token(r < nrows ? r : 0, hq);                  // (rows past the last one read the first)
        const u16* at = a.q + (c0 + (int64_t)t) * a.q_tok + (int64_t)hq * a.q_head + 16 * lg + 64 * (wave - KS * qt);
        wq[0] = gptr((const uint4_t*)at)[0];
        wq[1] = gptr((const uint4_t*)at)[1];
    }
    constexpr bool AHEAD = D == 256 && W == 4;                       // the next block's keys are fetched while this one's values are used
    if (AHEAD && j < nb) load_k(j);
    auto local_barrier = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    float* const qmax = (float*)(lds + QN * 2048);
    auto value = [&](int x) { return kv_value((u16)(wq[x >> 3][(x >> 1) & 3] >> (16 * (x & 1))), a.bf16); };
    if (wave < QN) {
        float mq = 0.f, bad = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            mq = fmaxf(mq, fabsf(value(x)));
            bad = __builtin_fmaf(value(x), 0.f, bad);                // NaN once a value is not finite
        }
        mq = fmaxf(mq, lane_xor(mq, 16, lane));
        mq = fmaxf(mq, lane_xor(mq, 32, lane));
        bad += lane_xor(bad, 16, lane);
        bad += lane_xor(bad, 32, lane);
        if (lg == 0) qmax[16 * wave + lr] = bad != 0.f ? bad : mq;
    }
    local_barrier();
    int E[RT], vend[RT];
    float qs[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float mq = 0.f, bad = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const float x = qmax[16 * (KS * rt + ks) + lr];
            mq = fmaxf(mq, x);
            bad = __builtin_isnan(x) ? x : bad;
        }
        if (bad != 0.f) mq = 1.f;                                    // the row's scores become NaN below
        E[rt] = mq > 0.f ? __builtin_amdgcn_frexp_expf(mq) : 0;
        qs[rt] = a.sl / QC + bad;
        const int r = row0 + 16 * rt + lr;
        vend[rt] = r < nrows ? sees(r / a.G) : 0;
    }
    if (wave < QN) {
        int e = E[0];
#pragma unroll
        for (int rt = 1; rt < RT; ++rt) e = qt == rt ? E[rt] : e;
        uint4_t dh, dl;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float f[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) f[y] = __builtin_fmaf(__builtin_amdgcn_ldexpf(value(4 * x + y), -e), QC, DIG);
            u32 hi, lo;
            digits(f[0], f[1], f[2], f[3], hi, lo);
            dh[x] = hi;
            dl[x] = lo;
        }
        ((uint4_t*)lds)[2 * wave * 64 + lane] = dh;
        ((uint4_t*)lds)[(2 * wave + 1) * 64 + lane] = dl;
    }
    local_barrier();
    const uint4_t* Q = (const uint4_t*)lds + lane;                   // digits hi, lo of K step ks of tile rt at 128 (KS rt + ks), + 64
    float4_t O[RT][DTL];
    float mr[RT], l[RT], u[RT];                                      // u: RT > 1, the row's outputs are in units of 2^u
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        mr[rt] = -__builtin_inff();
        l[rt] = 0.f;
        u[rt] = -160.f;                                              // (below every scale's)
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) O[rt][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    auto block = [&](auto edge) {
        if (!AHEAD) load_k(j);
        const float svj = sv;
        float c, f[16];                                              // one tile's scores at a time
        auto scores = [&](int rt) {
            c = __builtin_amdgcn_ldexpf(sk, E[rt]) * qs[rt];         // (the scales first: one may be huge where the other is tiny)
            int4_t hi[4], lo[4];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint4_t qh = Q[128 * (KS * rt + ks)], ql = Q[128 * (KS * rt + ks) + 64];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    hi[kt] = mma_i8(K[kt][ks], qh, ks ? hi[kt] : int4_t{0, 0, 0, 0});
                    lo[kt] = mma_i8(K[kt][ks], ql, ks ? lo[kt] : int4_t{0, 0, 0, 0});
                }
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) f[x] = (float)((hi[x >> 2][x & 3] << 8) + lo[x >> 2][x & 3]);
            if (rt == RT - 1) {
                __builtin_amdgcn_sched_barrier(0);                   // (the values' loads no earlier: they take the keys' registers)
                load_v(j);
                if (AHEAD && j + step < nb) load_k(j + step);
            }
        };
        auto left = [&](int rt, int x) { return 16 * (x >> 2) + (x & 3) < vend[rt] - j * KB - 4 * lg; };   // key x of this lane group is visible
        auto largest = [&](int rt) {
            if constexpr (edge)
#pragma unroll
                for (int x = 0; x < 16; ++x) f[x] = left(rt, x) ? f[x] : -__builtin_inff();
            float mx = f[0];
#pragma unroll
            for (int x = 1; x < 16; ++x) mx = fmaxf(mx, f[x]);
            return mx;
        };
        auto across = [&](float mx) {
            mx = fmaxf(mx, lane_xor(mx, 16, lane));
            return fmaxf(mx, lane_xor(mx, 32, lane));
        };
        if constexpr (RT == 1) {
            scores(0);
            const float mx = across(largest(0));
            const bool none = edge && mx == -__builtin_inff();       // the row sees no key of the block
            const float mb = none ? 0.f : mx * c;
            float p[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) p[x] = __builtin_amdgcn_exp2f((f[x] - mx) * c);   // at most 1: the digits hold no more (mb is rounded,
                                                                                            // f c - mb past zero from scores of some hundreds on)
            if constexpr (edge)                                      // also where c is 0, or nothing visible, and the product above NaN
#pragma unroll
                for (int x = 0; x < 16; ++x) p[x] = left(0, x) ? p[x] : 0.f;
            // the sum of the rounded probabilities, which are the weights that the values get: whole numbers in the low bits of p + DIG
            u32 lb = -16u * __float_as_uint(DIG);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                p[x] = __builtin_fmaf(p[x], PC, DIG);
                lb += __float_as_uint(p[x]);
            }
            uint4_t Ph, Pl;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                u32 h4, l4;
                digits(p[4 * x], p[4 * x + 1], p[4 * x + 2], p[4 * x + 3], h4, l4);
                Ph[x] = h4;
                Pl[x] = l4;
            }
            const bool up = !none && mb > mr[0] + 8.f;
            if (__builtin_amdgcn_ballot_w64(up)) {                   // uniform
                const float al = up ? __builtin_amdgcn_exp2f(mr[0] - mb) : 1.f;
                l[0] *= al;
#pragma unroll
                for (int dt = 0; dt < DTL; ++dt) O[0][dt] *= al;
                mr[0] = up ? mb : mr[0];
            }
            const float w = none ? 0.f : __builtin_amdgcn_exp2f(mb - mr[0]), be = none ? 0.f : w * (svj * (1.f / PC));
            l[0] = __builtin_fmaf(w * (1.f / PC), (float)(int)lb, l[0]);
#pragma unroll
            for (int dt = 0; dt < DTL; ++dt) {
                const int4_t z = {0, 0, 0, 0};
                const int4_t oh = mma_i8(V[dt], Ph, z), ol = mma_i8(V[dt], Pl, z);
#pragma unroll
                for (int e = 0; e < 4; ++e) O[0][dt][e] = __builtin_fmaf((float)((oh[e] << 8) + ol[e]), be, O[0][dt][e]);
            }
        } else {
            // the block's value scale 2^ls (the logarithm of the mantissa: that of a denormal scale itself would be taken as one of zero). A scale
            // of zero, which no append makes, counts as the smallest one.
            const float es = svj == 0.f ? -150.f : (float)__builtin_amdgcn_frexp_expf(svj);
            const float ls = svj == 0.f ? es : es + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(svj));
            half8_t P[RT][2], ones;
#pragma unroll
            for (int x = 0; x < 8; ++x) ones[x] = (_Float16)1.f;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                scores(rt);
                const float mx = largest(rt);
                // FP16 probabilities 2^(s - m + lu), whose products with the codes are in units of 2^u. (mr -inf: the row's first key)
                float lu = ls - u[rt], mz = lu - mr[rt], g = 1.f;
                bool cut = false;
                if (__builtin_amdgcn_ballot_w64(__builtin_fmaf(mx, c, mz) > 15.f || lu < 0.f)) {   // uniform
                    const float m0 = mr[rt], ma = across(mx), mb = edge && ma == -__builtin_inff() ? ma : ma * c;
                    const bool up = mb > m0 + 8.f;
                    const float down = up ? m0 - mb : 0.f;           // what the sums so far lie under the new maximum
                    mr[rt] = up ? mb : m0;
                    l[rt] *= __builtin_amdgcn_exp2f(down);
                    // a unit for the block's largest product where that is past FP16, one for the block's scale where the probabilities
                    // would fall out of it, as far as the outputs so far leave room for that (2^100)
                    float n = u[rt];
                    if (mb - mr[rt] + lu > 15.f) n = es - UP + fminf(__builtin_ceilf(mb - mr[rt]), 0.f);
                    if (__builtin_amdgcn_ballot_w64(ls < n)) {       // uniform
                        float mo = 0.f;
#pragma unroll
                        for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) mo = fmaxf(mo, fabsf(O[rt][dt][e]));
                        mo = across(mo);
                        const float room = mo > 0.f ? u[rt] + down + (float)(__builtin_amdgcn_frexp_expf(mo) - 100) : -__builtin_inff();
                        n = ls < n ? fminf(n, fmaxf(es - UP, room)) : n;
                    }
                    const float y = fmaxf(u[rt] - n + down, -500.f), yi = __builtin_floorf(y), yf = __builtin_amdgcn_exp2f(y - yi);
                    u[rt] = n;
                    lu = ls - n;
                    if (__builtin_amdgcn_ballot_w64(m0 != -__builtin_inff())) {           // uniform; else the outputs are zeros
#pragma unroll
                        for (int dt = 0; dt < DTL; ++dt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) O[rt][dt][e] = __builtin_amdgcn_ldexpf(O[rt][dt][e] * yf, (int)yi);
                    }
                    cut = __builtin_amdgcn_ballot_w64(lu < 0.f);
                    if (cut) {                                       // no room: the sum takes the probabilities all the same, the values'
                        g = lu < 0.f ? __builtin_amdgcn_exp2f(lu - UP) : 1.f;       // products of those rows lie below 2^-60 of their outputs
                        lu = lu < 0.f ? (float)UP : lu;
                    }
                    mz = lu - mr[rt];
                }
                if (edge && mr[rt] == -__builtin_inff()) mz = 0.f;
                float p[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(f[x], c, mz));
                if constexpr (edge)
#pragma unroll
                    for (int x = 0; x < 16; ++x) p[x] = left(rt, x) ? p[x] : 0.f;
#pragma unroll
                for (int x = 0; x < 16; ++x) P[rt][x >> 3][x & 7] = (_Float16)p[x];
                float4_t s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[rt][0], float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[rt][1], s, 0, 0, 0);
                l[rt] = __builtin_fmaf(s[0], __builtin_amdgcn_exp2f(-lu), l[rt]);        // (the same in all four lane groups)
                if (cut)                                             // uniform
#pragma unroll
                    for (int x = 0; x < 16; ++x) P[rt][x >> 3][x & 7] *= (_Float16)g;
            }
#pragma unroll
            for (int dt = 0; dt < DTL; ++dt) {
                half8_t A[2];
                widen(V[dt], A[0], A[1]);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) O[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[s], P[rt][s], O[rt][dt], 0, 0, 0);
            }
        }
        j += step;
    };
    const int whole = all / KB;                                      // blocks that every row sees whole (rows past the last one do not count)
    while (j < min(nb, whole)) block(std::false_type());
    while (j < nb) block(std::true_type());
    // merge the waves through LDS, a row tile at a time: statistics and outputs, wave w summing its share of the dim tiles
    constexpr int WD = DTL < W ? DTL : W, DW = DTL / WD;             // waves that sum, dim tiles of each
    float4_t* x = (float4_t*)lds;
    float *sm = (float*)(lds + W * DTL * 1024), *sl = sm + 16 * W;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        __syncthreads();
        float s = l[rt];
        if (RT == 1) {
            s += lane_xor(s, 16, lane);
            s += lane_xor(s, 32, lane);
        }
        if (lg == 0) {
            sm[16 * wave + lr] = mr[rt];
            sl[16 * wave + lr] = s;
        }
#pragma unroll
        for (int dt = 0; dt < DTL; ++dt) {
            float4_t y = O[rt][dt];
            if (RT > 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_ldexpf(y[e], (int)u[rt]);
            x[(wave * DTL + dt) * 64 + lane] = y;
        }
        __syncthreads();
        const int r = row0 + 16 * rt + lr;
        if (wave >= WD || r >= nrows) continue;
        float mx = -__builtin_inff(), lsum = 0.f, wt[W];
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, sm[16 * w + lr]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            // a wave without a visible key has l = 0 and weight 0; one whose scores are NaN has l = NaN and weight NaN
            const float mw = sm[16 * w + lr], lw = sl[16 * w + lr];
            wt[w] = mw == -__builtin_inff() ? lw : __builtin_amdgcn_exp2f(mw - mx);
            lsum = __builtin_fmaf(wt[w], lw, lsum);
        }
        int hq;
        const int t = token(r, hq);
        const size_t row = (size_t)(c0 + t) * (a.Hk * a.G) + hq;
        if (a.S > 1 && wave == 0 && lg == 0) {
            a.stat[(row * a.S + split) * 2] = mx;
            a.stat[(row * a.S + split) * 2 + 1] = lsum;
        }
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;            // a row that sees no key: zeros
#pragma unroll
        for (int k = 0; k < DW; ++k) {
            const int dt = wave * DW + k;
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float4_t y = x[(w * DTL + dt) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(wt[w], y[e], v[e]);
            }
            if (a.S > 1) *gptr((float4_t*)(a.part + (row * a.S + split) * D + 16 * dt + 4 * lg)) = v;
            else store4(a.o + row * D + 16 * dt + 4 * lg, v * inv, a.bf16);
        }
    }
}

// The splits' outputs of a row joined, weights exp2(m_s - max m). Few splits (at most 8): D / 4 threads a row, 4 dims each, every load at entry.
// A launch and two memory latencies: 256 rows x 8 parts x 128 4.8 us.
template <int D>
__global__ __launch_bounds__(KT) void k_kv8_join_few(KvAttend a) {
    constexpr int TD = D / 4, MS = 8;
    const int S = a.S, b = blockIdx.z, Hq = a.Hk * a.G, d = threadIdx.x % TD, i = blockIdx.x * (KT / TD) + threadIdx.x / TD, t = i / Hq;
    const int c0 = a.cu ? max(0, a.cu[b]) : b * a.most;
    if (t >= min(min(a.cu ? a.cu[b + 1] - c0 : a.most, a.most), a.rows - c0)) return;
    const size_t row = (size_t)(c0 + t) * Hq + (i - t * Hq);
    const float* pt = a.part + row * S * D + 4 * d;
    float2_t st[MS];
    float4_t v[MS];
#pragma unroll
    for (int s = 0; s < MS; ++s) {                           // (a split past the last reads that one again)
        st[s] = *gptr((const float2_t*)(a.stat + (row * S + min(s, S - 1)) * 2));
        v[s] = *gptr((const float4_t*)(pt + (size_t)min(s, S - 1) * D));
    }
    float mx = st[0].x, L = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 1; s < MS; ++s) mx = fmaxf(mx, st[s].x);
#pragma unroll
    for (int s = 0; s < MS; ++s) {                           // without a maximum: 0, or NaN
        const float w = s >= S ? 0.f : st[s].x == -__builtin_inff() ? st[s].y : __builtin_amdgcn_exp2f(st[s].x - mx);
        if (s < S) L = __builtin_fmaf(w, st[s].y, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = s < S ? __builtin_fmaf(w, v[s][e], acc[e]) : acc[e];
    }
    store4(a.o + row * D + 4 * d, acc * (L == 0.f ? 0.f : 1.f / L), a.bf16);
}

// More splits: grid (most x Hq, 1, B), one row a workgroup. The first wave works out the weights (lane = split) while thread (g, 4 dims) has
// its first eight of every (JT / (D / 4))th split under way. 16 rows x 128 parts x 256 4.0 us (with 256 threads 4.8).
constexpr int JT = 1024;         // its threads
template <int D>
__global__ __launch_bounds__(JT) void k_kv8_join(KvAttend a) {
    constexpr int TD = D / 4, NG = JT / TD, SR = MAX_SPLITS / 64, U = 8;
    __shared__ float4_t sums[NG][TD];
    __shared__ float wt[MAX_SPLITS], tot;
    const int tid = threadIdx.x, d = tid % TD, g = tid / TD, S = a.S, b = blockIdx.z, Hq = a.Hk * a.G, t = blockIdx.x / Hq;
    const int c0 = a.cu ? max(0, a.cu[b]) : b * a.most;
    if (t >= min(min(a.cu ? a.cu[b + 1] - c0 : a.most, a.most), a.rows - c0)) return;
    const size_t row = (size_t)(c0 + t) * Hq + (blockIdx.x - t * Hq);
    const float* st = a.stat + row * S * 2;
    const float* pt = a.part + row * S * D + 4 * d;
    float4_t v[U];
    auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < U; ++k)
            v[k] = s0 + g + k * NG < S ? *gptr((const float4_t*)(pt + (size_t)(s0 + g + k * NG) * D)) : float4_t{0.f, 0.f, 0.f, 0.f};
    };
    load(0);
    if (tid < 64) {
        float m[SR], l[SR], mx = -__builtin_inff(), L = 0.f;
#pragma unroll
        for (int r = 0; r < SR; ++r) {
            const int s = 64 * r + tid;
            m[r] = s < S ? gptr(st)[2 * s] : -__builtin_inff();
            l[r] = s < S ? gptr(st)[2 * s + 1] : 0.f;
            mx = fmaxf(mx, m[r]);
        }
        mx = wave_max(mx);
#pragma unroll
        for (int r = 0; r < SR; ++r) {
            const float x = m[r] == -__builtin_inff() ? l[r] : __builtin_amdgcn_exp2f(m[r] - mx);   // 0, or NaN, without a maximum
            wt[64 * r + tid] = x;
            L = __builtin_fmaf(x, l[r], L);
        }
        L = wave_sum(L);
        if (tid == 0) tot = L;
    }
    __syncthreads();
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += U * NG) {
        if (s0) load(s0);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int s = s0 + g + k * NG;
            const float x = s < S ? wt[s] : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(x, v[k][e], acc[e]);
        }
    }
    sums[g][d] = acc;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int k = 1; k < NG; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += sums[k][d][e];
    store4(a.o + row * D + 4 * d, acc * (tot == 0.f ? 0.f : 1.f / tot), a.bf16);
}

constexpr int64_t MAX_Z = 65535;  // the grid's z
size_t kv_attend_lds(int D, int W, int RT) {     // the waves' outputs and statistics of a row tile, or the query digits and maxima before them
    return max((size_t)W * ((D / 16) * 1024 + 128), (size_t)RT * (D / 64) * (2048 + 64));
}
bool kv_dim(int D) { return D == 64 || D == 128 || D == 256; }
bool kv_size(int B, int H, int nblk) { return B > 65535 || H > 65535 || nblk > (1 << 25) - 1; }

// How a call is split: the waves W of a workgroup, which take the blocks of 16 RT rows of a KV head in turn, and the parts S of their keys.
//   Two tiles of 16 rows a wave (D up to 128; 256 has no registers left for it) where that still makes two workgroups a CU: 2 x 1024 rows of
//   16 heads x 128 behind up to 4096 keys 93.5 us against 100.6, 4096 rows 95.8 against 106.2, 4 x 1024 rows of 16 heads x 64 25.7 against
//   28.9; with half as many workgroups it loses (968 rows of 16 x 128 13.8 against 12.7). Single rows of as many sequences go there too, by
//   the same rule, and are bound by memory either way: 64 sequences of 8 heads x 128 behind 4096 keys 96 against 99.5 (5.6 TB/s), 128 behind
//   1 to 2 thousand 76 against 74.
//   Few rows over up to 16 blocks: one launch of eight waves (50 rows of 4 sequences behind 800 keys, D = 256: 10.3 us against 12.6 in parts
//   of four waves with their join, 10 rows of 16 sequences 10.4 against 13.7; one row behind 968 9.9 against 8.9, but a call from Python
//   12 against 15.5).
//   Else four waves (968 causal rows of 8 heads x 256 13.5 us, with eight 17.0), in as many parts as give every CU a workgroup. Where that is
//   fewer than 4 and the parts stay long, as many as fit: the lengths of a batch differ (16 sequences of 4 to 8 thousand keys, 8 heads of
//   128: 44.3 us against 55.5).
//   (Times of calls one after the other in a captured graph, joins included.)
struct KvPlan {
    int W, S, RT;
};
KvPlan kv_plan(int B, int most, int G, int Hk, int D, int keys) {
    const int64_t n = (int64_t)most * G, heads = (int64_t)B * Hk, nb = ((int64_t)keys + KB - 1) / KB;
    if (D <= 128 && heads * ((n + 31) / 32) >= 512) return {4, 1, 2};
    const int64_t groups = heads * ((n + 15) / 16);
    if (groups <= 256 && nb <= 16) return {8, 1, 1};
    int64_t S = max((int64_t)1, min(256 / groups, (nb + 3) / 4));
    if (S < 4) S = max(S, min((D == 256 ? 512 : 1024) / groups, nb * D / 2048));
    return {4, (int)min(S, (int64_t)MAX_SPLITS), 1};
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
    const bool vec = !(((uintptr_t)k | (uintptr_t)v) % 16) && !((k_tok | k_head | v_tok | v_head) % 8);
    const KvAppend a = {(const u16*)k, (const u16*)v, k_tok, k_head, v_tok, v_head, cu, start, (i8*)k8, (i8*)v8, scale, (u16*)tail,
                        rows, most, H, D, nblk, max(k_tok, v_tok) < (1 << 24) && min(k_tok, v_tok) >= 0};
    const dim3 grid((u32)(2 * min((int64_t)nblk, ((int64_t)most + KB - 2) / KB + 1)), H, B);
    hipStream_t st = (hipStream_t)stream;
#define KV_APPEND(N)                                                                                    \
    do {                                                                                                \
        if (dtype == TCQ_BF16 && vec) launch_k(k_kv8_append<N, true, true>, grid, dim3(4 * N), 0, st, a);\
        else if (dtype == TCQ_BF16) launch_k(k_kv8_append<N, true, false>, grid, dim3(4 * N), 0, st, a); \
        else if (vec) launch_k(k_kv8_append<N, false, true>, grid, dim3(4 * N), 0, st, a);               \
        else launch_k(k_kv8_append<N, false, false>, grid, dim3(4 * N), 0, st, a);                       \
    } while (0)
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
#define KV_READ(N) launch_k(k_kv8_read<N>, dim3((u32)(2 * blocks * (N / 64)), H, B), dim3(KT), 0, (hipStream_t)stream, a)
    KV_BY_DIM(KV_READ);
#undef KV_READ
    return launch_status();
}

extern "C" int64_t tcq_kv8_attend_floats(int rows, int most, int B, int Hq, int Hk, int D, int keys) {
    if (rows <= 0 || most <= 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || keys < 0 || !kv_dim(D)) return 0;
    const int S = kv_plan(B, most, Hq / Hk, Hk, D, keys).S;
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
    const int G = Hq / Hk;
    const KvPlan plan = kv_plan(B, most, G, Hk, D, keys);
    const int S = plan.S;
    const int64_t tiles = ((int64_t)most * G + 16 * plan.RT - 1) / (16 * plan.RT);
    if ((int64_t)most * Hq > 0x7fffffff || (int64_t)rows * Hq > 0x7fffffff) return TCQ_ERR_UNSUPPORTED;
    if (S > 1 && !part) return TCQ_ERR_ARG;
    if (((uintptr_t)q | (uintptr_t)k8 | (uintptr_t)v8 | (uintptr_t)o | (uintptr_t)part) % 16 || (q_tok | q_head) % 8 || (uintptr_t)scale % 8)
        return TCQ_ERR_ALIGN;
    KvAttend a = {(const u16*)q, q_tok, q_head, cu, lens, (const i8*)k8, (const i8*)v8, scale, part, part + (S > 1 ? (size_t)rows * Hq * S * D : 0),
                  (u16*)o, score_scale * 1.44269504088896341f, rows, most, G, Hk, nblk, causal != 0, dtype == TCQ_BF16, S, 0};
    hipStream_t st = (hipStream_t)stream;
#define KV_ATTEND(N)                                                                                                    \
    do {                                                                                                                \
        const size_t lds = kv_attend_lds(N, plan.W, plan.RT);                                                           \
        for (int64_t left = tiles; left > 0; left -= MAX_Z) {                                                           \
            const dim3 grid((u32)(Hk * S), B, (u32)min(left, MAX_Z));                                                   \
            a.last = (int)(left - 1);                                                                                   \
            if (plan.W == 8) launch_k(k_kv8_attend<N, 8, 1>, grid, dim3(512), lds, st, a);                              \
            else if (N == 256 || plan.RT == 1) launch_k(k_kv8_attend<N, 4, 1>, grid, dim3(256), lds, st, a);            \
            else launch_k(k_kv8_attend<N == 64 ? 64 : 128, 4, 2>, grid, dim3(256), lds, st, a);                         \
            const int e = launch_status();                                                                              \
            if (e) return e;                                                                                            \
        }                                                                                                               \
        if (S > 1) {                                                                                                    \
            constexpr int PR = KT / (N / 4);                                                                            \
            if (S > 8) launch_k(k_kv8_join<N>, dim3((u32)most * Hq, 1, B), dim3(JT), 0, st, a);                         \
            else launch_k(k_kv8_join_few<N>, dim3(((u32)most * Hq + PR - 1) / PR, 1, B), dim3(KT), 0, st, a);             \
        }                                                                                                               \
    } while (0)
    KV_BY_DIM(KV_ATTEND);
#undef KV_ATTEND
    return launch_status();
}
