// Softmax attention of 16-bit query rows over key / value rows of 8 .. 256 dims, found through a page table (tcq_paged_attend) or in
// a batch of an encoder's states (tcq_cross_attend): o = softmax(scale q k^T) v, FP32 scores, statistics and outputs in one pass.
//
// Rows are (token, query head of the KV head's group). Scores are computed transposed, S^T = K Q^T, so that a lane's accumulators belong to one
// row: its maximum and sum need one exchange across lanes a tile, and the probabilities, rounded to 16 bits (the sum takes the rounded
// ones), are the right operand of O^T = V^T P^T where they are: the order in which the score product leaves the keys in a lane is the order in which
// the values are fetched, by transposing reads of their rows in LDS. Rows of keys and values go from memory to LDS directly, in 16-byte
// pieces whose place in the row is turned by the row's number so that the reads meet no bank twice.
//
// k_attend_rows, many rows: 32 rows a wave, so a wave reads every key and value of its tiles from LDS once for 32 rows: at 128 bytes a cycle that is as
// long as its products (bound: LDS reads and vector instructions, 144 and 32 exponentials for 32 products a tile of 64 keys x 128 dims). 64
// rows a wave would halve the reads, but leave one wave a SIMD (297 us for the case below at 235 to 250), eight waves a workgroup share the writes
// only (242), and scores of the next tile computed beside the exponentials of this one gain nothing while the reads bound both (260). (The times of that
// comparison took the maximum off inside the exponentials' multiply-add, 1 to 2 % less, 64 dims 5.) MI355X, calls in a row: 2 x 4096 rows of 16 heads x 128
// to up to 4096 states 236 to 246 us (980 to 1020 TFLOP/s; an 8192^3 product reaches 1260); to 4096 states, 8 heads x 256 1110 TFLOP/s, 32 x 64 880.
// At 256 dims 2 to 12 registers spill over pages and with a mask (a mask that hides a fifth of those keys saves no time: 249 us after 247; 8 x 968 causal
// rows of 8 heads on 1 x 256 in pages 65 us).
// k_attend_few, few rows: 16 rows a workgroup, four waves that share the keys; bound by memory from some MB on: 32 sequences of 16 heads on 8 x 128
// behind 4 to 8 thousand keys 149 us (814 MB, 5.5 TB/s), by latencies below (one row behind 968 keys 10.7 us with the join).
#include "tcq_device.h"
#include "tcq_launch.h"
#include "tcq_paged_rows.h"

#include <type_traits>

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// A probability is exp2((S - m) sl + LIFT), the difference first: S sl - m sl as one multiply-add with a rounded m sl is off by up to 2^-25 |m sl|, which
// from scores of about 10^7 on takes FP16 probabilities (10^9: BF16) out of their range and gives keys met before and after a new maximum different
// weights. The maximum follows for the same reason when S - m passes its step, not when S passes a rounded m + step.
// FP16 probabilities lie 2^7 higher (the maximum follows in steps of 2^8, so at most 2^15): those of 2^-21 of the largest keep all their digits
template <bool BF> constexpr float LIFT = BF ? 0.f : 7.f;
// The maximum of a row that has seen keys, all of them with scores of -inf. Maxima are of the products q k: times a scale above 0.78 it would be the
// -inf of a row that has seen none.
constexpr float LOWEST = -3.0e38f;

struct Attn {
    const u16* q;
    int64_t q_tok, q_head;               // elements
    const char *k, *v;
    int64_t kb, kh, kt, vb, vh, vt;      // bytes: page (or sequence), head, token
    const int* table;                    // pages: (B, N)
    const uint8_t* mask;                 // states: (B, T), mask_b apart
    int64_t mask_b;
    const int *cu, *lens;
    u16* o;
    float *part, *stat;                  // split: outputs (row, head, split, D) and maxima (of the products, not scaled) / sums (.., 2)
    int rows, most, Hk, G, D, N, shift, pages, cap, causal, S, tiles, sorted;
    float sl, step;                      // the scale to powers of two, and how far scores may pass the maximum before it follows: 2^8
};


template <bool BF>
__device__ __forceinline__ float16_t mma32(uint4_t a, uint4_t b, float16_t c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ float4_t mma16(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ float prob(float d, float sl) {
    return __builtin_amdgcn_exp2f(BF ? d * sl : __builtin_fmaf(d, sl, LIFT<BF>));
}
// two probabilities as 16-bit values, to nearest, and their sum as the values say: the weights that the values get add up to one. (16 bits are what the
// products take; a second product for the rest would double theirs. Relative error of an output against 64 bits 2.1e-3 in BF16, 2.8e-4
// in FP16, where its own rounding is 1.7e-3 and 2.1e-4.)
template <bool BF>
__device__ __forceinline__ u32 prob2(float a, float b) {
    return BF ? bf16_cvt2(a, b) : __builtin_bit_cast(u32, __builtin_convertvector(float2_t{a, b}, half2_t));
}
template <bool BF>
__device__ __forceinline__ float sum2(u32 w, float c) {
    if constexpr (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w), __builtin_bit_cast(half2_t, 0x3c003c00u), c, false);
}
// Values that are not finite: a causal row that does not see a later token's must not make 0 * inf of it. In tiles that rows see in part they count as
// zeros, and where there were any their rows are read again after the last tile, for the rows that see them.
// bit 15 (31) of the result: the low (high) half of w is no finite value
template <bool BF>
__device__ __forceinline__ u32 not_finite(u32 w) {
    return BF ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
// a fragment with zeros in their places; odd: whether there were any
template <bool BF>
__device__ __forceinline__ uint4_t finite(uint4_t w, u32& odd) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const u32 t = not_finite<BF>(w[x]);
        odd |= t;
        w[x] &= ~(t | (t - (t >> 15)));
    }
    return w;
}
// of four values those that are not finite
template <bool BF>
__device__ __forceinline__ float4_t odd_ones(uint2_t w) {
    float4_t v;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const u32 h = (w[x >> 1] >> (16 * (x & 1))) & 0xffffu;
        v[x] = not_finite<BF>(h) & 0x8000u ? (BF ? bf16_to_f32((u16)h) : f16_to_f32((u16)h)) : 0.f;
    }
    return v;
}
template <bool BF>
__device__ __forceinline__ u32 out2(float a, float b) {
    return BF ? bf16x2(a, b) : (u32)f32_to_f16(a) | ((u32)f32_to_f16(b) << 16);
}
// 4 x 16 transposing read: lane i of 16 gets column i of the rows that lanes 4 r .. 4 r + 3 name in 8-byte pieces
__device__ __forceinline__ uint2_t read_tr(const char* p) {
    return __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p));
}
// at most vm loads (63: any) and lgkm LDS operations (15: any) still under way
template <int vm, int lgkm>
__device__ __forceinline__ void wait_for() {
    __builtin_amdgcn_s_waitcnt((vm & 15) | ((vm >> 4) << 14) | (7 << 4) | (lgkm << 8));
}
__device__ __forceinline__ void order() { asm volatile("" ::: "memory"); }

// Rows of DP dims (RS bytes) in LDS: the 16-byte piece p of row r lies at p ^ turn(r) of its row. A quarter wave reads one piece of 16 keys, half a wave
// 64 bytes of 4 value rows (32 x 32 products: wide) or 32 bytes of 8 (16 x 16): no two on the same of the 64 banks.
template <int DP>
struct Place {
    static constexpr int RS = 2 * DP, PR = DP / 8, NI = PR / 4;          // bytes and pieces of a row, 1 KiB loads of 16 rows
    __device__ static int key(int r) { return DP == 64 ? (r >> 1) & 7 : DP == 96 ? (r >> 2) & 3 : r & 15; }
    __device__ static int wide(int r) { return DP == 64 ? (2 * r) & 4 : DP == 96 ? 0 : 4 * (r & 3); }
    __device__ static int val(int r) { return DP == 64 ? r & 6 : DP == 96 ? 0 : 2 * (r & 7); }
};

// What a workgroup's sequence is: its rows, keys and what its tokens see.
struct Seq {
    int64_t c0;
    int n, cnt, len, end;                // processed and all new tokens, keys held, keys counted
    __device__ __forceinline__ int sees(int t, int causal) const { return causal ? max(0, min(len, end - cnt + t + 1)) : len; }
};
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ Seq seq_of(const Attn& a, int b) {
    Seq s;
    const int64_t c0 = a.cu ? a.cu[b] : (int64_t)b * a.most;
    s.cnt = uniform(max(0, a.cu ? a.cu[b + 1] - (int)c0 : a.most));
    s.c0 = uniform((int)max((int64_t)0, min(c0, (int64_t)a.rows)));
    s.n = min(min(s.cnt, a.most), a.rows - (int)s.c0);
    s.end = uniform(a.lens ? a.lens[b] : a.cap);
    s.len = max(0, min(s.end, a.cap));
    return s;
}

// First byte of the 16 rows from key p on (a page's, or a sequence's) of keys and values. A table's entry outside the pool counts as page 0.
template <bool PAGED>
struct Rows {
    const int* tab;
    int64_t k0, v0;
    __device__ __forceinline__ Rows(const Attn& a, int b, int h) {
        tab = PAGED ? a.table + (int64_t)b * a.N : nullptr;
        k0 = h * a.kh + (PAGED ? 0 : b * a.kb);
        v0 = h * a.vh + (PAGED ? 0 : b * a.vb);
    }
    __device__ __forceinline__ int page(const Attn& a, int p) const {
        if constexpr (!PAGED) return 0;
        const int e = p < a.cap ? tab[p >> a.shift] : 0;
        return __builtin_amdgcn_readfirstlane((u32)e < (u32)a.pages ? e : 0);
    }
    __device__ __forceinline__ const char* key(const Attn& a, int p, int page) const {
        return a.k + k0 + (PAGED ? page * a.kb + (p & ((1 << a.shift) - 1)) * a.kt : p * a.kt);
    }
    __device__ __forceinline__ const char* val(const Attn& a, int p, int page) const {
        return a.v + v0 + (PAGED ? page * a.vb + (p & ((1 << a.shift) - 1)) * a.vt : p * a.vt);
    }
};
// 16 bytes a lane at its offset from a uniform base, zeros from `bytes` on. A token's row is no longer than the way to the next, so `bytes` of n
// rows cuts off whole rows: those behind the last key need no test of their own. (The compiler must see that a descriptor is the same for the
// wave, or it makes a loop over its lanes: hence uniform.)
__device__ __forceinline__ rsrc_t rows_rsrc(const char* base, u32 bytes) {
    const u64 p = (u64)base;
    return make_rsrc((const void*)((u64)(u32)uniform((int)p) | (u64)(u32)uniform((int)(p >> 32)) << 32), (u32)uniform((int)bytes));
}
__device__ __forceinline__ uint4_t row_piece(const char* base, u32 bytes, u32 off, int more) {
    return __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(base, bytes), off, more, 0));
}
__device__ __forceinline__ void row_to_lds(const char* base, u32 bytes, u32 off, char* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rows_rsrc(base, bytes), (__attribute__((address_space(3))) void*)dst, 16, off, 0, 0, 0);
}

__device__ __forceinline__ u64 first_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// Which tile of R rows of which sequence and head workgroup k takes: the k-th when they are ordered by the keys that they see (in steps of 64), the
// most first, so that the last ones to start are short. A lane counts for one sequence (at most 64); found by bisection of the number of keys.
struct Job {
    int b, h, tile;
};
__device__ __forceinline__ int wave_total(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);
    return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48);
}
__device__ __forceinline__ Job longest(const Attn& a, int B, int R, int k) {
    const int lane = threadIdx.x & 63, b = min(lane, B - 1);
    const int c0 = a.cu ? a.cu[b] : b * a.most, cnt = max(0, a.cu ? a.cu[b + 1] - c0 : a.most), at = max(0, min(c0, a.rows));
    const int n = lane < B ? min(min(cnt, a.most), a.rows - at) : 0, end = a.lens ? a.lens[b] : a.cap, len = max(0, min(end, a.cap));
    const int nrows = n * a.G, tiles = (nrows + R - 1) / R;
    // tiles of the sequence that see at least x keys: the tokens from x - end + cnt - 1 on do, tile i ends with row R (i + 1) - 1
    auto count = [&](int x) {
        if (x <= 0) return tiles;
        if (x > len) return 0;
        if (!a.causal) return tiles;
        const int t = max(0, x - end + cnt - 1);
        return t >= n ? 0 : tiles - t * a.G / R;
    };
    int lo = 0, hi = (a.cap >> 6) + 1;                                   // the most steps that more than k tiles see
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (wave_total(count(64 * mid)) * a.Hk > k) lo = mid;
        else hi = mid;
    }
    const int more = count(64 * (lo + 1)), same = count(64 * lo) - more;
    int left = k - wave_total(more) * a.Hk, before = same;              // among those of `lo` steps, by sequence
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(before, d);
        before += lane >= d ? y : 0;
    }
    before = (before - same) * a.Hk;
    const u64 mine = __builtin_amdgcn_ballot_w64(same > 0 && before <= left);
    if (left < 0 || !mine) return {0, 0, a.tiles};                       // (no such tile: past the rows of every sequence)
    const int who = 63 - __builtin_clzll(mine);
    left -= __builtin_amdgcn_readlane(before, who);
    if (left >= __builtin_amdgcn_readlane(same, who) * a.Hk) return {0, 0, a.tiles};
    return {who, left % a.Hk, __builtin_amdgcn_readlane(tiles - more, who) - 1 - left / a.Hk};
}

// ------------------------------------------------------------------------------------------------------------ many rows
constexpr int rows_keys(int DP) { return DP == 256 ? 32 : 64; }       // keys of a tile

// W waves of 32 rows each; tiles of BK keys and values in LDS, the next tile's loads in flight behind one barrier a tile. Scores and
// outputs on 32 x 32 x 16 products: row r of a wave is column r of S^T and O^T.
template <int DP, bool BF, bool PAGED, bool MASK, int W>
__global__ __launch_bounds__(64 * W, 2) void k_attend_rows(Attn a) {
    using P = Place<DP>;
    constexpr int BK = rows_keys(DP), NK = BK / 32, KS = DP / 16, DT = DP / 32, HALF = BK * P::RS;   // (a tile's values lie HALF behind its keys)
    constexpr int NG = BK / 16, U = 2 * NG / W;                          // units of 16 rows of keys, then values; those of a wave
    static_assert(U * W == 2 * NG, "every wave fetches as much");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h2 = lane >> 5, r32 = lane & 31;
    const int groups = gridDim.x / a.tiles, gi = blockIdx.x % groups;
    int s = 0, h, b, at_tile;
    if (a.sorted) {
        const Job x = longest(a, groups / a.Hk, 32 * W, blockIdx.x);
        b = x.b, h = x.h, at_tile = x.tile;
    } else {
        s = gi % a.S, h = gi / a.S % a.Hk, b = gi / a.S / a.Hk;
        at_tile = a.tiles - 1 - blockIdx.x / groups;
    }
    const Seq sq = seq_of(a, b);
    constexpr int RW = 32;                                               // rows of a wave
    const int nrows = sq.n * a.G, row0 = at_tile * RW * W;
    if (row0 >= nrows) return;
    // (tiles that are not full leave waves without rows: not always on the same SIMD)
    const int wrow = row0 + RW * ((wave + blockIdx.x + (blockIdx.x >> 8)) % W), smax = sq.sees((min(row0 + RW * W, nrows) - 1) / a.G, a.causal), nt = (smax + BK - 1) / BK;
    const int t0 = (int)((int64_t)nt * s / a.S), t1 = (int)((int64_t)nt * (s + 1) / a.S);
    const Rows<PAGED> at(a, b, h);

    // this lane's row: its place (row, head) in q and o, the keys that it sees, its query, 16 bytes of dims 16 ks + 8 h2 .. a K step
    const int row = wrow + r32, some = min(row, nrows - 1), tok = some / a.G, hq = h * a.G + some - tok * a.G;
    const int vend = row < nrows ? sq.sees(tok, a.causal) : 0;
    uint4_t Q[KS];
    {
        const u16* p = a.q + (sq.c0 + tok) * a.q_tok + hq * a.q_head + 8 * h2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) Q[ks] = 16 * ks + 8 * h2 < a.D ? *gptr((const uint4_t*)(p + 16 * ks)) : uint4_t{0, 0, 0, 0};
    }
    // A wave fetches U units of 16 rows of a tile, P::NI loads of 1 KiB each, piece L of the rows at 16 L in LDS. Keys that no row sees are zeros:
    // those behind the last one by the bound of the loads, masked ones (bits) lane by lane.
    const uint8_t* mrow = MASK ? a.mask + b * a.mask_b : nullptr;
    auto mask_byte = [&](int j) { return lane < BK && BK * j + lane < smax ? (int)gptr(mrow)[BK * j + lane] : 0; };
    u32 off[U][P::NI];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool val = W > NG ? wave >= NG : W * u >= NG;              // unit u of the wave holds values (uniform)
#pragma unroll
        for (int i = 0; i < P::NI; ++i) {
            const int L = 64 * i + lane, r = L / P::PR, p = (L - r * P::PR) ^ (val ? P::wide(r) : P::key(r));
            off[u][i] = 8 * p < a.D ? (u32)(r * (val ? a.vt : a.kt)) + 16 * p : RSRC_OOB;
        }
    }
    auto fetch = [&](int j, u64 bits, const int (&page)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool val = W > NG ? wave >= NG : W * u >= NG;
            const int g = (wave + W * u) % NG, p0 = BK * j + 16 * g;
            const char* const base = val ? at.val(a, p0, page[u]) : at.key(a, p0, page[u]);
            const u32 bytes = (u32)max(0, min(16, smax - p0)) * (u32)(val ? a.vt : a.kt);
            char* const dst = lds + (2 * (j & 1) + (int)val) * HALF + g * 16 * P::RS;
#pragma unroll
            for (int i = 0; i < P::NI; ++i) {
                u32 o = off[u][i];
                if constexpr (MASK) o = (u32)(bits >> (16 * g)) >> ((64 * i + lane) / P::PR) & 1 ? o : RSRC_OOB;
                row_to_lds(base, bytes, o, dst + i * 1024);
            }
        }
    };
    auto pages_of = [&](int j, int (&page)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) page[u] = at.page(a, BK * j + 16 * ((wave + W * u) % NG));
    };
    // byte offsets of the fragments in a tile: K step ks of the first 32 keys, dims 32 dt .. of the first 8 values (turns stay within 256 bytes)
    constexpr int FK = KS < 8 ? KS : 8, FV = DT < 4 ? DT : 4;
    int fk[FK], fv[FV];
#pragma unroll
    for (int ks = 0; ks < FK; ++ks) fk[ks] = r32 * P::RS + 16 * ((2 * ks + h2) ^ P::key(r32));
    {
        const int i = lane & 15, r = 4 * h2 + (i >> 2);
#pragma unroll
        for (int dt = 0; dt < FV; ++dt) fv[dt] = HALF + r * P::RS + 16 * ((4 * dt + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ P::wide(r)) + 8 * (i & 1);
    }
    float16_t O[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[dt][e] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    u32 odd = 0;

    int page[U], mb = 0;                                                 // pages of the next tile
    u64 b0 = 0, b1 = 0;                                                  // MASK: bits of tiles j, j + 1
    if (t0 < t1) {
        if (MASK) {
            b1 = __builtin_amdgcn_ballot_w64(mask_byte(t0) != 0);
            mb = mask_byte(t0 + 1);
        }
        pages_of(t0, page);
        fetch(t0, b1, page);
        pages_of(t0 + 1, page);
    }
    // One tile, the next one's loads under way. edge: rows may see a part of it.
    auto step = [&](int j, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        wait_for<0, 0>();                                                // this wave's rows in LDS, and its reads of the tile before
        order();
        __builtin_amdgcn_s_barrier();
        order();
        if (MASK) {
            b0 = b1;
            b1 = __builtin_amdgcn_ballot_w64(mb != 0);
            mb = mask_byte(j + 2);
        }
        if (j + 1 < t1) {
            fetch(j + 1, b1, page);
            pages_of(j + 2, page);
        }
        if (wrow >= nrows || (MASK && !b0)) return;                      // uniform: no rows, or no keys that count
        const char* T = lds + (j & 1) * 2 * HALF;
        float16_t S[NK];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) S[kt][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kt = 0; kt < NK; ++kt) S[kt] = mma32<BF>(*(const uint4_t*)(T + fk[ks % FK] + 256 * (ks / FK) + kt * 32 * P::RS), Q[ks], S[kt]);
        __builtin_amdgcn_s_setprio(0);                                   // (products before the other wave's vector instructions)
        float mx = LOWEST;
        if (EDGE && (!MASK || b0 != first_bits(BK))) {                   // uniform (a mask is the same for all rows)
            const u64 mine = MASK ? b0 : first_bits(min(BK, vend - BK * j));
            if (!mine) mx = -__builtin_inff();
            const u64 x = mine >> (4 * h2);
#pragma unroll
            for (int kt = 0; kt < NK; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    S[kt][e] = ((u32)(x >> (32 * kt)) >> (8 * (e >> 2) + (e & 3))) & 1 ? S[kt][e] : -__builtin_inff();
        }
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, S[kt][e]);
        mx = fmaxf(mx, lane_xor(mx, 32, lane));
        const bool up = mx - m > a.step;                                    // the maximum follows in steps: probabilities stay below 2^8
        if (__builtin_amdgcn_ballot_w64(up)) {                           // uniform
            const float al = up ? __builtin_amdgcn_exp2f((m - mx) * a.sl) : 1.f;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) O[dt] *= al;
            m = up ? mx : m;
        }
        const float mr = fmaxf(m, LOWEST);                               // (a row that has seen nothing yet: its scores are -inf)
        uint4_t Pr[2 * NK];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const u32 x = prob2<BF>(prob<BF>(S[kt][e] - mr, a.sl), prob<BF>(S[kt][e + 1] - mr, a.sl));
                l = sum2<BF>(x, l);
                Pr[2 * kt + (e >> 3)][(e >> 1) & 3] = x;
            }
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);                               // (the values' reads no earlier: they take the scores' registers)
#pragma unroll
        for (int c = 0; c < 2 * NK; ++c)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const char* p = T + fv[dt % FV] + 256 * (dt / FV) + c * 16 * P::RS;
                const uint2_t x = read_tr(p), y = read_tr(p + 8 * P::RS);
                uint4_t v = uint4_t{x[0], x[1], y[0], y[1]};
                if constexpr (EDGE && PAGED) v = finite<BF>(v, odd);
                O[dt] = mma32<BF>(v, Pr[c], O[dt]);
            }
    };
    // the tiles that all rows see in full, and those that they may see in part
    const int tf = MASK ? t0 : max(t0, min(t1, sq.sees(row0 / a.G, a.causal) / BK));
    for (int j = t0; j < tf; ++j) step(j, std::false_type{});
    for (int j = tf; j < t1; ++j) step(j, std::true_type{});
    if (PAGED && __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, false)) {   // uniform
        const int last = min(BK * t1, smax);
        for (int p = tf * BK; p < last; ++p) {
            const char* v = at.val(a, p, at.page(a, p)) + 8 * h2;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (p < vend && 32 * dt + 8 * e < a.D) {
                        const float4_t x = odd_ones<BF>(*gptr((const uint2_t*)(v + 64 * dt + 16 * e)));
#pragma unroll
                        for (int i = 0; i < 4; ++i) O[dt][4 * e + i] += x[i];
                        order();
                    }
        }
    }
    l += lane_xor(l, 32, lane);
    if (row >= nrows) return;                                            // (the lanes of a row go together)
    const int64_t out = (sq.c0 + tok) * (int64_t)(a.Hk * a.G) + hq;
    if (a.S > 1) {
        float* p = a.part + (out * a.S + s) * a.D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 32 * dt + 8 * e + 4 * h2;
                if (d < a.D) *gptr((float4_t*)(p + d)) = float4_t{O[dt][4 * e], O[dt][4 * e + 1], O[dt][4 * e + 2], O[dt][4 * e + 3]};
            }
        if (h2 == 0) *gptr((float2_t*)(a.stat + (out * a.S + s) * 2)) = float2_t{m, l};
        return;
    }
    const float inv = m == -__builtin_inff() && l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            u32 w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = out2<BF>(O[dt][e + 2 * x] * inv, O[dt][e + 2 * x + 1] * inv);
            const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            const int d = 32 * dt + 2 * e + 8 * h2;
            if (d < a.D) *gptr((uint4_t*)(a.o + out * a.D + d)) = uint4_t{x[0], y[0], x[1], y[1]};
        }
}

// ------------------------------------------------------------------------------------------------------------- few rows
// 16 rows a workgroup; its W waves take tiles of 32 keys in turn, each with LDS of its own for the values (no barrier), the keys straight
// from memory into 16 x 16 x 32 fragments; the waves' outputs meet in LDS.
template <int DP, bool BF, bool PAGED, int W>
__global__ __launch_bounds__(64 * W, DP == 256 ? 2 : 4) void k_attend_few(Attn a) {
    using P = Place<DP>;
    constexpr int KS = DP / 32, DT = DP / 16, OS = DP + 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, lr = lane & 15;
    const int groups = gridDim.x / a.tiles, gi = blockIdx.x % groups, rt = a.tiles - 1 - blockIdx.x / groups;
    const int s = gi % a.S, h = gi / a.S % a.Hk, b = gi / a.S / a.Hk;
    const Seq sq = seq_of(a, b);
    const int nrows = sq.n * a.G, row0 = rt * 16;
    if (row0 >= nrows) return;
    const int row = row0 + lr, tok = min(row, nrows - 1) / a.G, hq = h * a.G + min(row, nrows - 1) - tok * a.G;
    const int smax = sq.sees((min(row0 + 16, nrows) - 1) / a.G, a.causal), smin = sq.sees(row0 / a.G, a.causal), nt = (smax + 31) >> 5;
    const int vend = row < nrows ? sq.sees(tok, a.causal) : 0;
    const int t0 = (int)((int64_t)nt * s / a.S), t1 = (int)((int64_t)nt * (s + 1) / a.S);
    const Rows<PAGED> at(a, b, h);
    const uint8_t* mrow = !PAGED && a.mask ? a.mask + b * a.mask_b : nullptr;

    uint4_t Q[KS];
    {
        const u16* p = a.q + (sq.c0 + tok) * a.q_tok + hq * a.q_head + 8 * lg;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) Q[ks] = 32 * ks + 8 * lg < a.D ? *gptr((const uint4_t*)(p + 32 * ks)) : uint4_t{0, 0, 0, 0};
    }
    char* const T = lds + wave * 32 * P::RS;
    u32 ov[P::NI];
#pragma unroll
    for (int i = 0; i < P::NI; ++i) {
        const int L = 64 * i + lane, r = L / P::PR, p = L - r * P::PR, pv = p ^ P::val(r);
        ov[i] = 8 * pv < a.D ? (u32)(r * a.vt) + 16 * pv : RSRC_OOB;
    }
    const u32 ok = (u32)(lr * a.kt) + 16 * lg;
    constexpr int FV = DT < 8 ? DT : 8;                                  // (turns stay within 256 bytes)
    int fv[FV];                                                          // byte offsets of dims 16 dt .. of the first 16 values
    {
        const int r = 4 * lg + (lr >> 2);
#pragma unroll
        for (int dt = 0; dt < FV; ++dt) fv[dt] = r * P::RS + 16 * ((2 * dt + ((lr >> 1) & 1)) ^ P::val(r)) + 8 * (lr & 1);
    }
    const int j1 = min(smax, 32 * t1);                                   // (no keys past the last tile)
    uint4_t K[2][KS];
    // keys that no row sees are zeros: in pages, those behind the last one, by the bound of the loads; of states, bits says which, lane by lane
    auto bytes_of = [&](int p0, int64_t step) { return PAGED ? (u32)max(0, min(16, j1 - p0)) * (u32)step : 16 * (u32)step; };
    auto load_k = [&](int j, u32 bits, const int (&page)[2]) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* const base = at.key(a, 32 * j + 16 * g, page[g]);
            const u32 bytes = bytes_of(32 * j + 16 * g, a.kt), off = PAGED || (bits >> (16 * g + lr)) & 1 ? ok : RSRC_OOB;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) K[g][ks] = row_piece(base, bytes, 32 * ks + 8 * lg < a.D ? off : RSRC_OOB, 64 * ks);
        }
    };
    auto load_v = [&](int j, u32 bits, const int (&page)[2]) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* const base = at.val(a, 32 * j + 16 * g, page[g]);
            const u32 bytes = bytes_of(32 * j + 16 * g, a.vt);
#pragma unroll
            for (int i = 0; i < P::NI; ++i)
                row_to_lds(base, bytes, PAGED || (bits >> (16 * g + (64 * i + lane) / P::PR)) & 1 ? ov[i] : RSRC_OOB, T + g * 16 * P::RS + i * 1024);
        }
    };
    auto bits_of = [&](int j) -> u32 {                                   // keys of tile j < t1 that any row may see
        if (j >= t1) return 0;
        u32 in = (u32)first_bits(min(32, smax - 32 * j));
        if (!PAGED && mrow) in &= (u32)__builtin_amdgcn_ballot_w64(32 * j + (lane & 31) < smax && gptr(mrow)[32 * j + (lane & 31)] != 0);
        return in;
    };
    float4_t O[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) O[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    u32 odd = 0;
    int j = t0 + wave, page[2];
    u32 bits = bits_of(j);
#pragma unroll
    for (int g = 0; g < 2; ++g) page[g] = at.page(a, 32 * j + 16 * g);
    load_k(j, bits, page);
    for (; j < t1; j += W) {
        load_v(j, bits, page);
        order();
        float4_t S[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            S[g] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) S[g] = mma16<BF>(K[g][ks], Q[ks], S[g]);
        }
        const u32 now = bits;
        const int jn = j + W;                                            // (past the last tile the loads read zeros)
        bits = bits_of(j + W);
#pragma unroll
        for (int g = 0; g < 2; ++g) page[g] = at.page(a, 32 * jn + 16 * g);
        order();
        load_k(jn, bits, page);
        order();
        float mx = LOWEST;
        u32 mine = ~0u;
        if (now != ~0u || 32 * j + 32 > smin || vend == 0) {
            mine = PAGED ? (u32)first_bits(min(32, vend - 32 * j)) : vend > 32 * j ? now : 0u;
            if (!mine) mx = -__builtin_inff();
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[g][e] = (mine >> (16 * g + 4 * lg + e)) & 1 ? S[g][e] : -__builtin_inff();
        }
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, S[g][e]);
        mx = fmaxf(mx, lane_xor(mx, 16, lane));
        mx = fmaxf(mx, lane_xor(mx, 32, lane));
        const bool up = mx - m > a.step;
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float al = up ? __builtin_amdgcn_exp2f((m - mx) * a.sl) : 1.f;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) O[dt] *= al;
            m = up ? mx : m;
        }
        const float mr = fmaxf(m, LOWEST);
        uint4_t Pr;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            Pr[x] = prob2<BF>(prob<BF>(S[x >> 1][2 * (x & 1)] - mr, a.sl), prob<BF>(S[x >> 1][2 * (x & 1) + 1] - mr, a.sl));
            l = sum2<BF>(Pr[x], l);
        }
        wait_for<2 * KS, 15>();                                          // the values are there; the next keys may be under way
        order();
        if (PAGED && 32 * j + 32 > smin && smin < smax) {                // uniform: rows that see different keys of the tile
#pragma unroll 1
            for (int i = lane; i < 2 * 16 * P::PR; i += 64) ((uint4_t*)T)[i] = finite<BF>(((const uint4_t*)T)[i], odd);
            wait_for<63, 0>();
            order();
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const char* p = T + fv[dt % FV] + 256 * (dt / FV);
            const uint2_t x = read_tr(p), y = read_tr(p + 16 * P::RS);
            O[dt] = mma16<BF>(uint4_t{x[0], x[1], y[0], y[1]}, Pr, O[dt]);
        }
        wait_for<63, 0>();                                               // the next values take the place of these
        order();
    }
    wait_for<0, 0>();                                                    // no load into the LDS outlives its tile
    if (PAGED && __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, false)) {   // uniform
        for (int e = t0 + wave; e < t1; e += W)
            for (int p = max(32 * e, smin / 32 * 32); p < min(32 * e + 32, smax); ++p) {
                const char* v = at.val(a, p, at.page(a, p)) + 8 * lg;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    if (p < vend && 16 * dt + 4 * lg < a.D) {
                        O[dt] += odd_ones<BF>(*gptr((const uint2_t*)(v + 32 * dt)));
                        order();
                    }
            }
    }
    l += lane_xor(l, 16, lane);
    l += lane_xor(l, 32, lane);
    __syncthreads();
    float* const X = (float*)lds;                                        // (W, 16, OS) outputs, (W, 16, 2) maxima and sums
    float* const Y = X + W * 16 * OS;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *(float4_t*)(X + (wave * 16 + lr) * OS + 16 * dt + 4 * lg) = O[dt];
    if (lg == 0) *(float2_t*)(Y + (wave * 16 + lr) * 2) = float2_t{m, l};
    __syncthreads();
    const int D4 = a.D >> 2;
    for (int u = threadIdx.x; u < 16 * D4; u += 64 * W) {
        const int r = u / D4, d = 4 * (u - r * D4), rr = row0 + r;
        if (rr >= nrows) break;
        float M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, Y[(w * 16 + r) * 2]);
        float L = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = Y[(w * 16 + r) * 2], x = mw == -__builtin_inff() ? (M == mw ? 1.f : 0.f) : __builtin_amdgcn_exp2f((mw - M) * a.sl);
            L = __builtin_fmaf(x, Y[(w * 16 + r) * 2 + 1], L);
            v += *(const float4_t*)(X + (w * 16 + r) * OS + d) * x;
        }
        const int t = rr / a.G;
        const int64_t out = (sq.c0 + t) * (int64_t)(a.Hk * a.G) + h * a.G + rr - t * a.G;
        if (a.S > 1) {
            *gptr((float4_t*)(a.part + (out * a.S + s) * a.D + d)) = v;
            if (d == 0) *gptr((float2_t*)(a.stat + (out * a.S + s) * 2)) = float2_t{M, L};
        } else {
            v *= M == -__builtin_inff() && L == 0.f ? 0.f : 1.f / L;
            *gptr((uint2_t*)(a.o + out * a.D + d)) = uint2_t{out2<BF>(v[0], v[1]), out2<BF>(v[2], v[3])};
        }
    }
}

// The parts of a row joined: 64 threads for a row and head (4 dims each) and NG of them side by side over its parts, in workgroups of four waves or more; grid
// (rows, B). Weights first (they are few), then the parts' outputs, eight loads under way. (16 rows of 128 parts: 13 us with NG = 4.)
constexpr int MAX_PARTS = 128;       // NP = 2 a lane
template <bool BF, int NG>
__global__ __launch_bounds__(64 * (NG > 4 ? NG : 4)) void k_attend_join(Attn a) {
    constexpr int NW = NG > 4 ? NG : 4;
    __shared__ float4_t sums[NW][64];
    const Seq sq = seq_of(a, blockIdx.y);
    const int Hq = a.Hk * a.G, d = threadIdx.x & 63, wave = threadIdx.x >> 6, g = wave % NG;
    static_assert(NG == 1 || NG == NW, "the waves that meet at the barrier have one row: they leave together");
    const int64_t out = join_row(sq.c0, sq.n, Hq, (int64_t)blockIdx.x * (NW / NG) + wave / NG);
    if (out < 0) return;                                                 // (before the loads: behind the rows the workspace ends)
    const bool on = 4 * d < a.D;
    const float* st = a.stat + out * a.S * 2;
    const float* p = a.part + out * a.S * a.D + 4 * d;
    constexpr int NP = NG == 1 ? 1 : MAX_PARTS / 64;                     // parts d, d + 64 of the row
    float mi[NP], li[NP], M = -__builtin_inff(), L = 0.f;
#pragma unroll
    for (int r = 0; r < NP; ++r) {
        const bool in = 64 * r + d < a.S;
        const float2_t x = in ? *gptr((const float2_t*)(st + 2 * (64 * r + d))) : float2_t{-__builtin_inff(), 0.f};
        mi[r] = x[0];
        li[r] = x[1];
        M = fmaxf(M, mi[r]);
    }
    M = wave_max(M);
    float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < NP; ++r) {
        const float w = mi[r] == -__builtin_inff() ? (M == mi[r] ? 1.f : 0.f) : __builtin_amdgcn_exp2f((mi[r] - M) * a.sl);
        L = __builtin_fmaf(w, li[r], L);
#pragma unroll 8
        for (int i = g; i < min(64, a.S - 64 * r); i += NG) {
            const float wi = lane_value(w, i);
            if (on) v += *gptr((const float4_t*)(p + (int64_t)(64 * r + i) * a.D)) * wi;
        }
    }
    L = wave_sum(L);
    if constexpr (NG > 1) {
        sums[wave][d] = v;
        __syncthreads();
        if (g) return;
#pragma unroll
        for (int k = 1; k < NG; ++k) v += sums[wave + k][d];
    }
    if (!on) return;
    v *= M == -__builtin_inff() && L == 0.f ? 0.f : 1.f / L;
    *gptr((uint2_t*)(a.o + out * a.D + 4 * d)) = uint2_t{out2<BF>(v[0], v[1]), out2<BF>(v[2], v[3])};
}

// How a call is split: which kernel, and the parts S of the keys (tiles of 64 of them).
//   Few rows: up to 32 of a KV head (its 16-row workgroups read every key once, or twice), and calls whose rows make no more than 320 such workgroups
//   over at most 16 tiles: their four waves share the keys of a row, where the other kernel would need parts and their join (50 rows of 32 heads x 48 to
//   600 keys 6.6 us against 10.0, 300 x 300 of 16 x 64 7.1 against 10.4, 8 x 50 rows of 8 heads on 1 x 256 behind 850 22.9 against 27.4; 4000 keys 83
//   against 46).
//   Parts: as many as fill the chip (at most 128), of one tile (the other kernel: two) or more. Few rows take 1024 workgroups (32 sequences of 16 heads on 8 x 128 behind
//   4 to 8 thousand keys 176 us, 512: 203, 2048: 179), but 16 and more rows a workgroup, whose parts are larger to write and to join, 512 over many
//   tiles (4 x 16 rows behind 8000 keys 42.6, 1024: 53) and 256 over few. No parts where they save less than their join takes, about 4 us, at
//   D / 200 us a tile.
//   (Times in a captured graph, joins included.)
struct Plan {
    int few, S;
};
Plan plan_of(int B, int most, int G, int Hk, int D, int keys) {
    const int64_t n = (int64_t)most * G, heads = (int64_t)B * Hk, tiles = ((int64_t)keys + 63) / 64;
    const bool few = n <= 32 || (heads * ((n + 15) / 16) <= 320 && tiles <= 16);
    const int64_t groups = heads * (few ? (n + 15) / 16 : (n + 127) / 128);
    const int64_t want = !few ? 512 : n < 16 ? 1024 : tiles >= 64 ? 512 : 256;
    int64_t S = max((int64_t)1, min(min(want / groups, tiles / (few && n < 16 ? 1 : 2)), (int64_t)MAX_PARTS));
    if (few && (tiles - tiles / S) * D < 800) S = 1;
    return {few, (int)S};
}
int64_t floats_of(int rows, int most, int B, int Hq, int Hk, int D, int keys) {
    if (rows <= 0 || most <= 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || keys < 0 || D <= 0 || D > 256 || D % 8) return 0;
    const int S = plan_of(B, most, Hq / Hk, Hk, D, keys).S;
    return S > 1 ? (int64_t)rows * Hq * S * (D + 2) : 0;
}

template <int DP, bool BF, bool PAGED>
int run_dim(Attn& a, const Plan& p, int B, hipStream_t st) {
    const int64_t n = (int64_t)a.most * a.G;
    if (p.few) {
        a.tiles = (int)((n + 15) / 16);
        const dim3 grid((u32)((int64_t)a.tiles * a.S * a.Hk * B));
        constexpr int W = 4;
        const size_t lds = max((size_t)W * 32 * Place<DP>::RS, (size_t)W * 16 * (DP + 4 + 2) * 4);
        launch_k(k_attend_few<DP, BF, PAGED, W>, grid, dim3(64 * W), lds, st, a);
    } else {
        constexpr int W = 4;
        a.tiles = (int)((n + 32 * W - 1) / (32 * W));
        const int64_t grid = (int64_t)a.tiles * a.S * a.Hk * B;
        const size_t lds = (size_t)4 * rows_keys(DP) * Place<DP>::RS;
        a.sorted = a.S == 1 && B <= 64 && grid > 512 && (a.causal || B > 1);
        if (!PAGED && a.mask) launch_k(k_attend_rows<DP, BF, false, true, W>, dim3((u32)grid), dim3(64 * W), lds, st, a);
        else launch_k(k_attend_rows<DP, BF, PAGED, false, W>, dim3((u32)grid), dim3(64 * W), lds, st, a);
    }
    return launch_status();
}

int run(Attn& a, bool bf, bool paged, int B, int keys, float* part, hipStream_t st) {
    const int Hq = a.Hk * a.G;
    const Plan p = plan_of(B, a.most, a.G, a.Hk, a.D, keys);
    a.S = p.S;
    if (a.S > 1 && !part) return TCQ_ERR_ARG;
    if ((uintptr_t)part % 16) return TCQ_ERR_ALIGN;
    a.part = part;
    a.stat = a.S > 1 ? part + (size_t)a.rows * Hq * a.S * a.D : nullptr;
    int e = 0;
#define ATTEND(N)                                                                                                          \
    e = paged ? (bf ? run_dim<N, true, true>(a, p, B, st) : run_dim<N, false, true>(a, p, B, st))                          \
              : (bf ? run_dim<N, true, false>(a, p, B, st) : run_dim<N, false, false>(a, p, B, st))
    if (a.D <= 64) ATTEND(64);
    else if (a.D <= 96) ATTEND(96);
    else if (a.D <= 128) ATTEND(128);
    else ATTEND(256);
#undef ATTEND
    if (e || a.S <= 1) return e;
    const int64_t rows = (int64_t)a.most * Hq;
#define JOIN(NG)                                                                                                        \
    do {                                                                                                                \
        constexpr int NW = NG > 4 ? NG : 4;                                                                             \
        const dim3 grid((u32)((rows + NW / NG - 1) / (NW / NG)), B);                                                    \
        if (bf) launch_k(k_attend_join<true, NG>, grid, dim3(64 * NW), 0, st, a);                                       \
        else launch_k(k_attend_join<false, NG>, grid, dim3(64 * NW), 0, st, a);                                         \
    } while (0)
    if (a.S > 32) JOIN(16);
    else if (a.S > 8) JOIN(4);
    else JOIN(1);
#undef JOIN
    return launch_status();
}

// The scale is above 0 and finite, so that 0 * -inf and 0 * inf do not come up (scores times 2^-149 are all 0); a first maximum passes the step whatever
// the scale.
void scale_of(Attn& a, float score_scale) {
    a.sl = fminf(fmaxf(score_scale * 1.44269504088896341f, 0x1p-149f), __FLT_MAX__);
    a.step = fminf(8.f / a.sl, __FLT_MAX__);
}

constexpr int64_t MANY = 0x7fffffff;
// what both attentions ask of their arguments
int refuse(const void* q, int64_t q_tok, int64_t q_head, int dtype, const int32_t* cu, int rows, int most, int B, int Hq, int Hk, int D, const void* k,
           int64_t kb, int64_t kh, int64_t kt, const void* v, int64_t vb, int64_t vh, int64_t vt, float score_scale, int keys, const void* o) {
    if (!q || !k || !v || !o || rows <= 0 || most <= 0 || B <= 0 || Hq <= 0 || Hk <= 0 || D <= 0 || keys < 0 || !(score_scale >= 0.f && score_scale < __builtin_inff()))
        return TCQ_ERR_ARG;
    if (dtype != TCQ_BF16 && dtype != TCQ_F16) return TCQ_ERR_DTYPE;
    if (Hq % Hk || (!cu && (int64_t)most * B > rows)) return TCQ_ERR_SHAPE;
    if (D > 256 || D % 8 || B > 65535 || Hk > 65535) return TCQ_ERR_UNSUPPORTED;
    if (min(min(min(q_tok, q_head), min(kb, kh)), min(min(kt, vb), min(vh, vt))) < 0 || max(kt, vt) >= (1 << 25) || min(kt, vt) < D) return TCQ_ERR_UNSUPPORTED;
    const int64_t n = (int64_t)most * (Hq / Hk);
    if (n > MANY - 256 || (int64_t)rows * Hq > MANY || (n / 16 + 1) * 64 * Hk > MANY / B || (int64_t)most * Hq > MANY) return TCQ_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 16 || (q_tok | q_head | kb | kh | kt | vb | vh | vt) % 8) return TCQ_ERR_ALIGN;
    return 0;
}

}  // namespace

extern "C" int64_t tcq_paged_attend_floats(int rows, int most, int B, int Hq, int Hk, int D, int keys) { return floats_of(rows, most, B, Hq, Hk, D, keys); }

extern "C" int tcq_paged_attend(const void* q, int64_t q_tok, int64_t q_head, int dtype, const int32_t* cu, const int32_t* lens, int rows, int most,
                                int B, int Hq, int Hk, int D, const void* k, int64_t k_page, int64_t k_head, int64_t k_tok, const void* v,
                                int64_t v_page, int64_t v_head, int64_t v_tok, int pages, int page_rows, const int32_t* table, int per_seq, int causal,
                                float score_scale, int keys, float* part, void* o, tcq_stream_t stream) {
    int e = refuse(q, q_tok, q_head, dtype, cu, rows, most, B, Hq, Hk, D, k, k_page, k_head, k_tok, v, v_page, v_head, v_tok, score_scale, keys, o);
    if (e) return e;
    if (!lens || !table || pages <= 0 || per_seq <= 0) return TCQ_ERR_ARG;
    if (page_rows < 16 || (page_rows & (page_rows - 1)) || page_rows > (1 << 20) || (int64_t)page_rows * per_seq > (1 << 30)) return TCQ_ERR_UNSUPPORTED;
    Attn a = {};
    a.q = (const u16*)q, a.q_tok = q_tok, a.q_head = q_head;
    a.k = (const char*)k, a.v = (const char*)v;
    a.kb = 2 * k_page, a.kh = 2 * k_head, a.kt = 2 * k_tok, a.vb = 2 * v_page, a.vh = 2 * v_head, a.vt = 2 * v_tok;
    a.table = table, a.cu = cu, a.lens = lens, a.o = (u16*)o;
    a.rows = rows, a.most = most, a.Hk = Hk, a.G = Hq / Hk, a.D = D, a.N = per_seq, a.shift = 31 - __builtin_clz(page_rows), a.pages = pages;
    a.cap = page_rows * per_seq, a.causal = causal != 0;
    scale_of(a, score_scale);
    return run(a, dtype == TCQ_BF16, true, B, min(keys, a.cap), part, (hipStream_t)stream);
}

extern "C" int64_t tcq_cross_attend_floats(int rows, int most, int B, int Hq, int Hk, int D, int keys) { return floats_of(rows, most, B, Hq, Hk, D, keys); }

extern "C" int tcq_cross_attend(const void* q, int64_t q_tok, int64_t q_head, int dtype, const int32_t* cu, int rows, int most, int B, int Hq, int Hk, int D,
                                const void* k, int64_t k_seq, int64_t k_head, int64_t k_tok, const void* v, int64_t v_seq, int64_t v_head, int64_t v_tok,
                                int keys, const int32_t* lens, const uint8_t* mask, int64_t mask_seq, float score_scale, float* part, void* o,
                                tcq_stream_t stream) {
    int e = refuse(q, q_tok, q_head, dtype, cu, rows, most, B, Hq, Hk, D, k, k_seq, k_head, k_tok, v, v_seq, v_head, v_tok, score_scale, keys, o);
    if (e) return e;
    if (keys <= 0) return TCQ_ERR_ARG;
    if (keys > (1 << 30)) return TCQ_ERR_UNSUPPORTED;
    Attn a = {};
    a.q = (const u16*)q, a.q_tok = q_tok, a.q_head = q_head;
    a.k = (const char*)k, a.v = (const char*)v;
    a.kb = 2 * k_seq, a.kh = 2 * k_head, a.kt = 2 * k_tok, a.vb = 2 * v_seq, a.vh = 2 * v_head, a.vt = 2 * v_tok;
    a.mask = mask, a.mask_b = mask_seq, a.cu = cu, a.lens = lens, a.o = (u16*)o;
    a.rows = rows, a.most = most, a.Hk = Hk, a.G = Hq / Hk, a.D = D, a.cap = keys;
    scale_of(a, score_scale);
    return run(a, dtype == TCQ_BF16, false, B, keys, part, (hipStream_t)stream);
}
