// Softmax attention of 16-bit query rows over key / value rows of 8 .. 256 dims, found through a page table (tcq_paged_attend) or in
// a batch of an encoder's states (tcq_cross_attend): o = softmax(scale q k^T) v, FP32 scores, statistics and outputs in one pass.
//
// Rows are (token, query head of the KV head's group). Scores are computed transposed, S^T = K Q^T, so that a lane's accumulators belong to one
// row: its maximum and sum need one exchange across lanes a tile, and the probabilities, rounded to 16 bits (the sum takes the rounded
// ones), are the right operand of O^T = V^T P^T where they are: the order in which the score product leaves the keys in a lane is the order in which
// the values are fetched, by transposing reads of their rows in LDS. Rows of keys and values go from memory to LDS directly, in 16-byte
// pieces whose place in the row is turned by the row's number so that the reads meet no bank twice.
#include "tcq_device.h"
#include "tcq_launch.h"

#include <type_traits>

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// FP16 probabilities lie 2^7 higher (the maximum follows in steps of 2^8, so at most 2^15): those of 2^-21 of the largest keep all their digits
template <bool BF> constexpr float LIFT = BF ? 0.f : 7.f;
constexpr float LOWEST = -3.0e38f;       // the maximum of a row that has seen keys, all of them with scores of -inf

struct Attn {
    const u16* q;
    int64_t q_tok, q_head;               // elements
    const char *k, *v;
    int64_t kb, kh, kt, vb, vh, vt;      // bytes: page (or sequence), head, token
    const int* table;                    // pages: (B, N)
    const uint8_t* mask;                      // states: (B, T), mask_b apart
    int64_t mask_b;
    const int *cu, *lens;
    u16* o;
    float *part, *stat;                  // split: outputs (row, head, split, D) and maxima / sums (.., 2)
    int rows, most, Hk, G, D, N, shift, pages, cap, causal, S, tiles;
    float sl;
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
// two probabilities as 16-bit values, and their sum as the values say. FP16 rounds towards zero (one instruction): the sum
// takes the same values, so the shift cancels and what remains is as large as that of the nearest ones.
template <bool BF>
__device__ __forceinline__ u32 prob2(float a, float b) {
    return BF ? bf16_cvt2(a, b) : __builtin_bit_cast(u32, __builtin_amdgcn_cvt_pkrtz(a, b));
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

// Rows of DP dims (RS bytes) in LDS: where the 16-byte piece p of key row r lies in its row. Keys are read 32 (16) rows at one piece,
// values 4 rows at one pair of pieces a quarter wave.
template <int DP>
struct Place {
    static constexpr int RS = 2 * DP, PR = DP / 8, NI = PR / 4;          // bytes and pieces of a row, 1 KiB loads of 16 rows
    __device__ static int key(int r) { return DP == 64 ? (r >> 1) & 7 : DP == 96 ? (r >> 2) & 3 : r & 15; }
    __device__ static int val(int r) { return DP == 64 ? (r & 6) : DP == 96 ? 0 : 2 * (r & 7); }
};

// What a workgroup's sequence is: its rows, keys and what its tokens see.
struct Seq {
    int64_t c0;
    int n, cnt, len, end;                // processed and all new tokens, keys held, keys counted
    __device__ __forceinline__ int sees(int t, int causal) const { return causal ? max(0, min(len, end - cnt + t + 1)) : len; }
};
__device__ __forceinline__ Seq seq_of(const Attn& a, int b) {
    Seq s;
    s.c0 = a.cu ? a.cu[b] : (int64_t)b * a.most;
    s.cnt = a.cu ? a.cu[b + 1] - (int)s.c0 : a.most;
    s.c0 = max((int64_t)0, min(s.c0, (int64_t)a.rows));
    s.cnt = max(0, s.cnt);
    s.n = (int)min((int64_t)min(s.cnt, a.most), a.rows - s.c0);
    s.end = a.lens ? a.lens[b] : a.cap;
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
constexpr u32 SPAN = 0x7ffffff0u;        // 16 rows from a base lie below 2 GiB
// 16 bytes a lane at its offset from a uniform base: to LDS (lane l at dst + 16 l), or to registers
__device__ __forceinline__ void row_to_lds(const char* base, u32 off, char* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(base, SPAN), (__attribute__((address_space(3))) void*)dst, 16, off, 0, 0, 0);
}
__device__ __forceinline__ uint4_t row_piece(const char* base, u32 off, int more) {
    return __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(base, SPAN), off, more, 0));
}

__device__ __forceinline__ u64 first_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// ------------------------------------------------------------------------------------------------------------ many rows
constexpr int rows_keys(int DP) { return DP == 256 ? 32 : 64; }      // keys of a tile

// W waves of 32 rows each; tiles of BK keys and values in LDS, the next tile's loads in flight behind one barrier a tile. Scores and
// outputs on 32 x 32 x 16 products: row r of a wave is column r of S^T and O^T.
template <int DP, bool BF, bool PAGED, int W>
__global__ __launch_bounds__(64 * W, 2) void k_attend_rows(Attn a) {
    using P = Place<DP>;
    constexpr int BK = rows_keys(DP), NK = BK / 32, KS = DP / 16, DT = DP / 32, HALF = BK * P::RS;   // (a tile's values lie HALF behind its keys)
    constexpr int NG = BK / 16, NU = 2 * NG / W;                         // groups of 16 keys, and loads of 16 rows a wave
    static_assert(2 * NG % W == 0, "every wave loads as much");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h2 = lane >> 5, r32 = lane & 31;
    const int groups = gridDim.x / a.tiles, gi = blockIdx.x % groups, rt = a.tiles - 1 - blockIdx.x / groups;
    const int s = gi % a.S, h = gi / a.S % a.Hk, b = gi / a.S / a.Hk;
    const Seq sq = seq_of(a, b);
    const int nrows = sq.n * a.G, row0 = rt * 32 * W;
    if (row0 >= nrows) return;
    const int wrow = row0 + 32 * wave, row = wrow + r32, tok = min(row, nrows - 1) / a.G, hq = h * a.G + min(row, nrows - 1) - tok * a.G;
    const int smax = sq.sees((min(row0 + 32 * W, nrows) - 1) / a.G, a.causal), nt = (smax + BK - 1) / BK;
    const int wmax = wrow < nrows ? sq.sees((min(wrow + 32, nrows) - 1) / a.G, a.causal) : 0;
    const int vend = row < nrows ? sq.sees(tok, a.causal) : 0;
    const int t0 = (int)((int64_t)nt * s / a.S), t1 = (int)((int64_t)nt * (s + 1) / a.S);
    const Rows<PAGED> at(a, b, h);

    // the row's query, 16 bytes of dims 16 ks + 8 h2 .. a K step
    uint4_t Q[KS];
    {
        const u16* p = a.q + (sq.c0 + tok) * a.q_tok + hq * a.q_head + 8 * h2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) Q[ks] = 16 * ks + 8 * h2 < a.D ? *gptr((const uint4_t*)(p + 16 * ks)) : uint4_t{0, 0, 0, 0};
    }
    // offsets of this lane's pieces of 16 rows: piece L of the 16 rows' lies in LDS at 16 L
    u32 ok[P::NI], ov[P::NI];
#pragma unroll
    for (int i = 0; i < P::NI; ++i) {
        const int L = 64 * i + lane, r = L / P::PR, p = L - r * P::PR, pk = p ^ P::key(r), pv = p ^ P::val(r);
        ok[i] = 8 * pk < a.D ? (u32)(r * a.kt) + 16 * pk : RSRC_OOB;
        ov[i] = 8 * pv < a.D ? (u32)(r * a.vt) + 16 * pv : RSRC_OOB;
    }
    const uint8_t* mrow = !PAGED && a.mask ? a.mask + b * a.mask_b : nullptr;
    auto mask_byte = [&](int j) { return lane < BK && BK * j + lane < smax ? (int)gptr(mrow)[BK * j + lane] : 0; };
    // tile j's rows that some row sees (bits) to LDS; the others, which no row sees, are zeros there
    auto issue = [&](int j, int buf, u64 bits, const int (&page)[NU]) {
        if (!bits) return;
#pragma unroll
        for (int x = 0; x < NU; ++x) {
            const int u = wave + W * x, g = u % NG, p0 = BK * j + 16 * g;
            const bool val = W <= NG ? W * x >= NG : u >= NG;            // uniform
            char* dst = lds + buf * 2 * HALF + u * 16 * P::RS;
            const u32 on = (u32)(bits >> (16 * g)) & 0xffffu;
            const char* const base = val ? at.val(a, p0, page[x]) : at.key(a, p0, page[x]);
            if (on == 0xffffu) {
#pragma unroll
                for (int i = 0; i < P::NI; ++i)
                    row_to_lds(base, val ? ov[i] : ok[i], dst + i * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < P::NI; ++i)
                    row_to_lds(base, (on >> ((64 * i + lane) / P::PR)) & 1 ? (val ? ov[i] : ok[i]) : RSRC_OOB, dst + i * 1024);
            }
        }
    };
    auto pages_of = [&](int j, int (&page)[NU]) {
#pragma unroll
        for (int x = 0; x < NU; ++x) page[x] = at.page(a, BK * j + 16 * ((wave + W * x) % NG));
    };
    // byte offsets of the fragments in a tile: K step ks of the first 32 keys, dims 32 dt .. of the first 8 values (turns stay within 256 bytes)
    constexpr int FK = KS < 8 ? KS : 8, FV = DT < 4 ? DT : 4;
    int fk[FK], fv[FV];
#pragma unroll
    for (int ks = 0; ks < FK; ++ks) fk[ks] = r32 * P::RS + 16 * ((2 * ks + h2) ^ P::key(r32));
    {
        const int i = lane & 15, r = 4 * h2 + (i >> 2);
#pragma unroll
        for (int dt = 0; dt < FV; ++dt) fv[dt] = HALF + r * P::RS + 16 * ((4 * dt + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ P::val(r)) + 8 * (i & 1);
    }
    float16_t O[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[dt][e] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    u32 odd = 0;
    const float thr = 8.f / a.sl;

    int page[NU], mb = 0;
    u64 next = 0;
    auto bits_of = [&](int j) -> u64 {                                   // (mb: the mask's bytes of tile j)
        const u64 in = first_bits(min(BK, smax - BK * j));
        return !PAGED && mrow ? in & __builtin_amdgcn_ballot_w64(mb != 0) : in;
    };
    if (t0 < t1) {
        pages_of(t0, page);
        if (!PAGED && mrow) mb = mask_byte(t0);
        next = bits_of(t0);
        if (!PAGED && mrow) mb = mask_byte(t0 + 1);
        issue(t0, 0, next, page);
        pages_of(t0 + 1, page);
    }
    auto step = [&](int j, auto edge) {                                  // edge: rows may see a part of the tile
        constexpr bool EDGE = decltype(edge)::value;
        const int buf = (j - t0) & 1;
        const u64 bits = next;
        wait_for<0, 0>();                                                // this tile's loads, and the reads of the one before
        order();
        __builtin_amdgcn_s_barrier();
        order();
        if (j + 1 < t1) {
            next = bits_of(j + 1);
            if (!PAGED && mrow) mb = mask_byte(j + 2);
            issue(j + 1, buf ^ 1, next, page);
            pages_of(j + 2, page);
        }
        const char* T = lds + buf * 2 * HALF;
        if (EDGE ? !bits || BK * j >= wmax : wrow >= nrows) return;      // uniform
        float16_t S[NK];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt) {
#pragma unroll
            for (int e = 0; e < 16; ++e) S[kt][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) S[kt] = mma32<BF>(*(const uint4_t*)(T + fk[ks % FK] + 256 * (ks / FK) + kt * 32 * P::RS), Q[ks], S[kt]);
        }
        float mx = LOWEST;
        if constexpr (EDGE) {
            const u64 mine = PAGED ? first_bits(min(BK, vend - BK * j)) : vend > BK * j ? bits : 0ull;
            if (!mine) mx = -__builtin_inff();
            const u64 w = mine >> (4 * h2);
#pragma unroll
            for (int kt = 0; kt < NK; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    S[kt][e] = ((u32)(w >> (32 * kt)) >> (8 * (e >> 2) + (e & 3))) & 1 ? S[kt][e] : -__builtin_inff();
        }
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, S[kt][e]);
        mx = fmaxf(mx, lane_xor(mx, 32, lane));
        const bool up = mx > m + thr;                                    // the maximum follows in steps: probabilities stay below 2^8
        if (__builtin_amdgcn_ballot_w64(up)) {                           // uniform
            const float al = up ? __builtin_amdgcn_exp2f((m - mx) * a.sl) : 1.f;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) O[dt] *= al;
            m = up ? mx : m;
        }
        const float mc = fmaxf(m * a.sl, -__FLT_MAX__) - LIFT<BF>;       // (a row that has seen nothing yet: its scores are -inf)
        uint4_t Pr[2 * NK];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const u32 w = prob2<BF>(__builtin_amdgcn_exp2f(__builtin_fmaf(S[kt][e], a.sl, -mc)), __builtin_amdgcn_exp2f(__builtin_fmaf(S[kt][e + 1], a.sl, -mc)));
                l = sum2<BF>(w, l);
                Pr[2 * kt + (e >> 3)][(e >> 1) & 3] = w;
            }
        __builtin_amdgcn_sched_barrier(0);                               // (the values' reads no earlier: they take the scores' registers)
        auto values = [&](int c, int dt) {
            const char* p = T + fv[dt % FV] + 256 * (dt / FV) + c * 16 * P::RS;
            const uint2_t x = read_tr(p), y = read_tr(p + 8 * P::RS);
            return uint4_t{x[0], x[1], y[0], y[1]};
        };
#pragma unroll
        for (int c = 0; c < 2 * NK; ++c)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if constexpr (EDGE && PAGED) O[dt] = mma32<BF>(finite<BF>(values(c, dt), odd), Pr[c], O[dt]);
                else O[dt] = mma32<BF>(values(c, dt), Pr[c], O[dt]);
            }
    };
    // the tiles that all rows see in full, and those that they may see in part
    const int tf = !PAGED && mrow ? t0 : max(t0, min(t1, sq.sees(row0 / a.G, a.causal) / BK));
    for (int j = t0; j < tf; ++j) step(j, std::false_type{});
    for (int j = tf; j < t1; ++j) step(j, std::true_type{});
    if (PAGED && __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, false)) {   // uniform
        const int last = min(BK * t1, wmax);
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
    if (row >= nrows) return;
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
        if (h2 == 0) *gptr((float2_t*)(a.stat + (out * a.S + s) * 2)) = float2_t{m * a.sl, l};
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
    int orow[P::NI];
#pragma unroll
    for (int i = 0; i < P::NI; ++i) {
        const int L = 64 * i + lane, r = L / P::PR, p = L - r * P::PR, pv = p ^ P::val(r);
        orow[i] = r;
        ov[i] = 8 * pv < a.D ? (u32)(r * a.vt) + 16 * pv : RSRC_OOB;
    }
    const u32 ok = (u32)(lr * a.kt) + 16 * lg;
    int fv[DT];
    {
        const int r = 4 * lg + (lr >> 2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) fv[dt] = r * P::RS + 16 * ((2 * dt + ((lr >> 1) & 1)) ^ P::val(r)) + 8 * (lr & 1);
    }
    uint4_t K[2][KS];
    auto load_k = [&](int j, u32 bits, const int (&page)[2]) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* const base = at.key(a, 32 * j + 16 * g, page[g]);
            const u32 off = (bits >> (16 * g + lr)) & 1 ? ok : RSRC_OOB;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) K[g][ks] = row_piece(base, 32 * ks + 8 * lg < a.D ? off : RSRC_OOB, 64 * ks);
        }
    };
    auto load_v = [&](int j, u32 bits, const int (&page)[2]) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* const base = at.val(a, 32 * j + 16 * g, page[g]);
#pragma unroll
            for (int i = 0; i < P::NI; ++i)
                row_to_lds(base, (bits >> (16 * g + orow[i])) & 1 ? ov[i] : RSRC_OOB, T + g * 16 * P::RS + i * 1024);
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
    const float thr = 8.f / a.sl;
    int j = t0 + wave, page[2];
    u32 bits = bits_of(j);
#pragma unroll
    for (int g = 0; g < 2; ++g) page[g] = j < t1 ? at.page(a, 32 * j + 16 * g) : 0;
    load_k(j < t1 ? j : 0, bits, page);
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
        const int jn = j + W < t1 ? j + W : 0;                           // (past the last tile the loads read zeros)
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
        const bool up = mx > m + thr;
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float al = up ? __builtin_amdgcn_exp2f((m - mx) * a.sl) : 1.f;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) O[dt] *= al;
            m = up ? mx : m;
        }
        const float mc = fmaxf(m * a.sl, -__FLT_MAX__) - LIFT<BF>;
        uint4_t Pr;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            Pr[x] = prob2<BF>(__builtin_amdgcn_exp2f(__builtin_fmaf(S[x >> 1][2 * (x & 1)], a.sl, -mc)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(S[x >> 1][2 * (x & 1) + 1], a.sl, -mc)));
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
            const uint2_t x = read_tr(T + fv[dt]), y = read_tr(T + fv[dt] + 16 * P::RS);
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
    if (lg == 0) *(float2_t*)(Y + (wave * 16 + lr) * 2) = float2_t{m * a.sl, l};
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
            const float mw = Y[(w * 16 + r) * 2], x = mw == -__builtin_inff() ? (M == mw ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mw - M);
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

// The parts of a row joined: thread (row and head, 4 dims), grid (most * Hq * D / 4 threads, B).
template <bool BF>
__global__ __launch_bounds__(256) void k_attend_join(Attn a) {
    const Seq sq = seq_of(a, blockIdx.y);
    const int D4 = a.D >> 2, Hq = a.Hk * a.G;
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, x = u / D4;
    if (x >= (int64_t)sq.n * Hq) return;
    const int d = 4 * (int)(u - x * D4);
    const int64_t out = sq.c0 * Hq + x;
    const float* st = a.stat + out * a.S * 2;
    const float* p = a.part + out * a.S * a.D + d;
    float M = -__builtin_inff(), L = 0.f;
    for (int i = 0; i < a.S; ++i) M = fmaxf(M, gptr(st)[2 * i]);
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < a.S; ++i) {
        const float mi = gptr(st)[2 * i], w = mi == -__builtin_inff() ? (M == mi ? 1.f : 0.f) : __builtin_amdgcn_exp2f(mi - M);
        L = __builtin_fmaf(w, gptr(st)[2 * i + 1], L);
        v += *gptr((const float4_t*)(p + (int64_t)i * a.D)) * w;
    }
    v *= M == -__builtin_inff() && L == 0.f ? 0.f : 1.f / L;
    *gptr((uint2_t*)(a.o + out * a.D + d)) = uint2_t{out2<BF>(v[0], v[1]), out2<BF>(v[2], v[3])};
}

struct Plan {
    int few, S;
};
Plan plan_of(int B, int most, int G, int Hk, int D, int keys) {
    const int64_t n = (int64_t)most * G, heads = (int64_t)B * Hk;
    const int few = n <= 32;
    const int64_t groups = heads * (few ? (n + 15) / 16 : (n + 127) / 128), tiles = ((int64_t)keys + 63) / 64;
    const int64_t want = few ? 1024 : 512;
    const int64_t S = max((int64_t)1, min(min(want / groups, tiles / (few ? 4 : 4)), (int64_t)64));
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
        constexpr int W = 4;
        a.tiles = (int)((n + 15) / 16);
        const size_t lds = max((size_t)W * 32 * Place<DP>::RS, (size_t)W * 16 * (DP + 4 + 2) * 4);
        launch_k(k_attend_few<DP, BF, PAGED, W>, dim3((u32)((int64_t)a.tiles * a.S * a.Hk * B)), dim3(64 * W), lds, st, a);
    } else {
        constexpr int W = 4;
        a.tiles = (int)((n + 32 * W - 1) / (32 * W));
        launch_k(k_attend_rows<DP, BF, PAGED, W>, dim3((u32)((int64_t)a.tiles * a.S * a.Hk * B)), dim3(64 * W), (size_t)4 * rows_keys(DP) * Place<DP>::RS, st, a);
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
    const dim3 grid((u32)(((int64_t)a.most * Hq * (a.D / 4) + 255) / 256), B);
    if (bf) launch_k(k_attend_join<true>, grid, dim3(256), 0, st, a);
    else launch_k(k_attend_join<false>, grid, dim3(256), 0, st, a);
    return launch_status();
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
    if (min(min(min(q_tok, q_head), min(kb, kh)), min(min(kt, vb), min(vh, vt))) < 0 || max(kt, vt) >= (1 << 25)) return TCQ_ERR_UNSUPPORTED;
    const int64_t n = (int64_t)most * (Hq / Hk);
    if (n > MANY - 256 || (int64_t)rows * Hq > MANY || (n / 16 + 1) * 64 * Hk > MANY / B || (n * Hk / 256 + 1) * (D / 4) > MANY) return TCQ_ERR_UNSUPPORTED;
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
    a.sl = fmaxf(score_scale * 1.44269504088896341f, 1e-30f);
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
    a.sl = fmaxf(score_scale * 1.44269504088896341f, 1e-30f);
    return run(a, dtype == TCQ_BF16, false, B, keys, part, (hipStream_t)stream);
}
