// A pool of pages of key / value rows that sequences share: rows into pages, and the pool's bookkeeping on the device (which pages a
// sequence holds, how many sequences hold a page, which are free), so that a captured step takes its pages by itself.
//
// Every choice of a page is the lowest free one, for the sequences in their order: what a call does follows from its inputs alone. One
// workgroup makes the plan (the free pages are a bit each: 160000 pages are 20 KB), a grid of workgroups then copies the pages that the plan names, whose number
// only the device knows. Bookkeeping is bound by latency: a launch and a few dependent trips to memory; copies by memory. MI355X: room for 16 of 18
// sequences, each with a page copied, 5.6 us and 6.3 for the copies in 18 layers (38 MB, 6 TB/s, in part from the last-level cache), a fork of 16
// 3.9, a cut 3.5; compaction of 378 pages in 18 layers 5 + 79 us (453 MB, 5.7 TB/s); 9000 rows of 8 heads x 128 into pages 14.1 us
// (78 MB, 5.5 TB/s), 64 single rows 3.1.
#include "tcq_device.h"
#include "tcq_launch.h"

namespace {

// exclusive sums of two counts over the workgroup (T threads) in the order of the threads, and their totals; red: 16 pairs of LDS, free again after the
// next barrier
struct Two {
    int a, b;
};
template <int T>
__device__ __forceinline__ Two block_scan(Two v, Two* red, Two& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Two x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int p = __shfl_up(x.a, d), q = __shfl_up(x.b, d);
        x.a += lane >= d ? p : 0;
        x.b += lane >= d ? q : 0;
    }
    __syncthreads();
    if (lane == 63) red[wave] = x;
    __syncthreads();
    Two before = {0, 0}, sum = {0, 0};
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        before.a += w < wave ? red[w].a : 0;
        before.b += w < wave ? red[w].b : 0;
        sum.a += red[w].a;
        sum.b += red[w].b;
    }
    total = sum;
    return {before.a + x.a - v.a, before.b + x.b - v.b};
}

struct Book {
    int *table, *lens, *refs;
    u32* free;
    int* lack;
    int B, N, pages, words, T;
    // pages that n rows take, at most what a sequence has entries for
    __device__ __forceinline__ int held(int n) const { return (int)min(((int64_t)max(n, 0) + T - 1) / T, (int64_t)N); }
    __device__ __forceinline__ bool page(int p) const { return (u32)p < (u32)pages; }
    // the bits of word w that stand for pages
    __device__ __forceinline__ u32 valid(int w) const { return 32 * w + 32 <= pages ? ~0u : (1u << (pages - 32 * w)) - 1; }
    // one sequence less holds page p; without any it is free
    __device__ __forceinline__ void drop(int p) const {
        if (page(p) && atomicSub(refs + p, 1) == 1) atomicOr(free + (p >> 5), 1u << (p & 31));
    }
};

// Room for take[b] more rows of every sequence. moves: [0] the pages to copy, then their sources and destinations (B each).
// A sequence whose last page is partly filled and held by others gets a page of its own in its place. Served are the sequences in order
// as long as the pages last; the others stay as they are, start included, and count in lack.
// A thread for every page taken: with the pages of one word of the bits left to one thread 16 copies took 10.5 us instead of 5.6. 256 threads where that
// is one for every sequence and every 32 pages (11.9 us with 1024 and the pages left to one thread).
template <int PT>
__global__ __launch_bounds__(PT) void k_pages_take(Book a, const int* take, int* start, int* moves) {
    extern __shared__ int lds[];
    int* const off = lds;                                                  // (B) first of the pages a sequence takes, in the order of all
    int* const slot = lds + a.B;                                           // (B) its first new entry; bit 30: a copy of the page there
    __shared__ Two red[PT / 64];
    __shared__ int copies, served, missing, got[PT];
    const int tid = threadIdx.x;
    if (tid == 0) copies = served = missing = 0;
    u32 bits = tid < a.words ? a.free[tid] & a.valid(tid) : 0;                            // the first sweep's word; the others are only counted yet
    int rest = 0;
    for (int w = tid + PT; w < a.words; w += PT) rest += __popc(a.free[w] & a.valid(w));
    Two total, carry = {0, 0};
    int avail = 0, rank = 0;
    if (a.words > PT) {
        (void)block_scan<PT>({rest, 0}, red, total);
        avail = total.a;
    }
    for (int b0 = 0; b0 < a.B; b0 += PT) {
        const int b = b0 + tid;
        int need = 0, have = 0, copy = 0, len = 0, more = 0;
        bool fits = true;
        if (b < a.B) {
            len = max(0, a.lens[b]);
            more = max(0, take[b]);
            have = a.held(len);
            fits = (int64_t)len + more <= (int64_t)a.N * a.T;
            if (more && fits) {
                const int last = have && len % a.T ? a.table[(int64_t)b * a.N + have - 1] : -1;
                copy = a.page(last) && a.refs[last] > 1;
                need = a.held(len + more) - have + copy;
            }
        }
        const Two x = block_scan<PT>({need, b0 ? 0 : (int)__popc(bits)}, red, total);
        if (b0 == 0) {
            rank = x.b;
            avail += total.b;
            carry.b = total.b;
        }
        const int first = carry.a + x.a;
        carry.a += total.a;
        if (b < a.B) {
            const bool ok = fits && (need == 0 || first + need <= avail);
            off[b] = first;
            slot[b] = (have - copy) | (copy ? 1 << 30 : 0);
            start[b] = len;
            if (ok) {
                if (more) a.lens[b] = len + more;
                if (need) atomicMax(&served, first + need);
            } else if (more) atomicAdd(&missing, 1);
        }
    }
    __syncthreads();
    if (tid == 0 && missing) a.lack[0] += missing;
    const int want = served;
    for (int w0 = 0, done = 0; done < want; w0 += PT) {                    // (there are as many free pages: the loop ends)
        const int w = w0 + tid;
        int k = rank;
        if (w0) {
            bits = w < a.words ? a.free[w] & a.valid(w) : 0;
            const Two x = block_scan<PT>({(int)__popc(bits), 0}, red, total);
            k = done + x.a;
            done += total.a;
        } else done = carry.b;
        const u32 had = bits;
        // this sweep's pages of ranks c0 .. c0 + PT - 1 into LDS, then a thread for each
        for (int c0 = w0 ? done - total.a : 0; c0 < min(done, want); c0 += PT) {
            for (; bits && k < min(want, c0 + PT); ++k, bits &= bits - 1) got[k - c0] = 32 * w + __ffs(bits) - 1;
            __syncthreads();
            const int r = c0 + tid;
            if (r < min(done, want)) {
                const int p = got[tid];
                int lo = 0, hi = a.B;                                      // the last sequence whose pages start at r or before
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (off[mid] <= r) lo = mid;
                    else hi = mid;
                }
                int* const e = a.table + (int64_t)lo * a.N + (slot[lo] & ~(1 << 30)) + r - off[lo];
                if (r == off[lo] && slot[lo] >> 30) {
                    const int i = atomicAdd(&copies, 1);                   // (the order of the copies changes nothing)
                    moves[1 + i] = *e;
                    moves[1 + a.B + i] = p;
                }
                *e = p;
                a.refs[p] = 1;
            }
            __syncthreads();
        }
        if (bits != had) atomicAnd(a.free + w, ~(had ^ bits));             // (the copied pages' words take atomics below)
        if (w0 + PT >= a.words) break;
    }
    __syncthreads();
    const int n = copies;
    for (int i = tid; i < n; i += PT) a.drop(moves[1 + i]);
    if (tid == 0) moves[0] = n;
}

// grid n: sequence dst[i], which holds nothing, holds the pages and rows of src[i]. Pairs that name no sequence, the same one, one that holds rows as
// dst, a dst that an earlier pair names or any pair's dst as src are left out and count in lack.
__global__ __launch_bounds__(256) void k_pages_fork(Book a, const int* src, const int* dst, int n) {
    const int i = blockIdx.x, s = src[i], d = dst[i];
    const bool in = (u32)s < (u32)a.B && (u32)d < (u32)a.B && s != d && a.lens[d] <= 0;
    int bad = !in;
    for (int j = threadIdx.x; j < n; j += 256) bad |= (j < i && dst[j] == d) || dst[j] == s;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicAdd(a.lack, 1);
        return;
    }
    const int len = max(0, a.lens[s]), held = a.held(len);
    for (int j = threadIdx.x; j < held; j += 256) {
        const int p = a.table[(int64_t)s * a.N + j];
        a.table[(int64_t)d * a.N + j] = p;
        if (a.page(p)) atomicAdd(a.refs + p, 1);
    }
    if (threadIdx.x == 0) a.lens[d] = len;
}

// grid B: sequence b keeps its first keep[b] rows and gives back the pages behind them
__global__ __launch_bounds__(64) void k_pages_trim(Book a, const int* keep) {
    const int b = blockIdx.x, len = max(0, a.lens[b]), end = max(0, min(len, keep[b]));
    const int h0 = a.held(end), h1 = a.held(len);
    for (int j = h0 + threadIdx.x; j < h1; j += 64) {
        int* const e = a.table + (int64_t)b * a.N + j;
        a.drop(*e);
        *e = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) a.lens[b] = end;
}

// The plan of a compaction: U pages are in use; the i-th of them from page U on moves to the i-th free one below U. moves: [0] how many, [1] U, then
// sources and destinations (pages / 2 each) and the new places of all pages that move (pages).
template <int PT>
__global__ __launch_bounds__(PT) void k_pages_plan(Book a, int* moves) {
    __shared__ Two red[PT / 64];
    const int tid = threadIdx.x, half = a.pages / 2;
    int free = 0;
    for (int w = tid; w < a.words; w += PT) free += __popc(a.free[w] & a.valid(w));
    Two total, carry = {0, 0};
    (void)block_scan<PT>({free, 0}, red, total);
    const int U = a.pages - total.a;
    int *const src = moves + 2, *const dst = src + half, *const to = dst + half;
    for (int w0 = 0; w0 < a.words; w0 += PT) {
        const int w = w0 + tid;
        u32 low = 0, high = 0;
        if (w < a.words) {
            const u32 f = a.free[w] & a.valid(w), below = 32 * w + 32 <= U ? ~0u : 32 * w >= U ? 0u : (1u << (U - 32 * w)) - 1;
            low = f & below;
            high = ~f & a.valid(w) & ~below;
            if (low | high) a.free[w] = a.valid(w) & ~below;
        }
        const Two x = block_scan<PT>({(int)__popc(high), (int)__popc(low)}, red, total);
        int i = carry.a + x.a, k = carry.b + x.b;
        carry.a += total.a;
        carry.b += total.b;
        for (; high; high &= high - 1) src[i++] = 32 * w + __ffs(high) - 1;
        for (; low; low &= low - 1) dst[k++] = 32 * w + __ffs(low) - 1;
    }
    __syncthreads();
    for (int i = tid; i < carry.a; i += PT) {
        const int s = src[i], d = dst[i];
        to[s] = d;
        a.refs[d] = a.refs[s];
        a.refs[s] = 0;
    }
    if (tid == 0) {
        moves[0] = carry.a;
        moves[1] = U;
    }
}

// Pages copied in all layers of keys and values, 16 KiB of one at a time; the table's entries of pages that moved are renamed by the first workgroups.
constexpr int CHUNK = 16384;
struct Copy {
    char *k, *v;
    int64_t page, layer;               // bytes
    int layers, pages;
    const int *count, *src, *dst;      // count NULL: n pairs
    int n;
    int *table, entries;               // renamed: entries >= *from, by to
    const int *from, *to;
};
__global__ __launch_bounds__(256) void k_pages_copy(Copy a) {
    const int n = a.count ? min(*a.count, a.n) : a.n;
    if (n <= 0) return;
    if (a.table) {
        const int U = *a.from;
        for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < a.entries; e += (int64_t)gridDim.x * 256) {
            const int p = a.table[e];
            if (p >= U && p < a.pages && (u32)a.to[p] < (u32)U) a.table[e] = a.to[p];
        }
    }
    const int64_t per = (a.page + CHUNK - 1) / CHUNK, units = per * n * a.layers * 2;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t c = u % per, x = u / per;
        const int i = (int)(x % n), lv = (int)(x / n), l = lv >> 1, s = a.src[i], d = a.dst[i];
        if ((u32)s >= (u32)a.pages || (u32)d >= (u32)a.pages || s == d) continue;
        char* const base = (lv & 1 ? a.v : a.k) + l * a.layer + c * CHUNK + threadIdx.x * 16;
        const int64_t left = a.page - c * CHUNK - threadIdx.x * 16;
        uint4_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q * 4096 < left) w[q] = *gptr((const uint4_t*)(base + s * a.page + q * 4096));
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q * 4096 < left) *gptr((uint4_t*)(base + d * a.page + q * 4096)) = w[q];
    }
}

struct Append {
    const u16 *k, *v;
    int64_t kt, kh, vt, vh;            // elements
    u16 *pk, *pv;
    int64_t kp, kph, kpt, vp, vph, vpt;
    const int *table, *lens, *start, *cu;
    int rows, most, H, D, N, shift, pages;
};
// grid (pieces of most rows, B): row i of sequence b goes to position start[b] + i. A thread takes E values of the keys and of the values.
template <int E>
__global__ __launch_bounds__(256) void k_pages_append(Append a) {
    const int b = blockIdx.y, per = a.H * a.D / E;
    int64_t c0 = a.cu ? a.cu[b] : (int64_t)b * a.most;
    const int cnt = a.cu ? a.cu[b + 1] - (int)c0 : a.most;
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int i = (int)(u / per), x = (int)(u - (int64_t)i * per), h = x / (a.D / E), d = E * (x - h * (a.D / E));
    if (i >= min(cnt, a.most) || c0 < 0 || c0 + i >= a.rows) return;
    const int64_t pos = (int64_t)a.start[b] + i;
    if (pos < 0 || pos >= a.lens[b] || pos >= (int64_t)a.N << a.shift) return;
    const int p = a.table[(int64_t)b * a.N + (pos >> a.shift)];
    if ((u32)p >= (u32)a.pages) return;
    const int64_t t = pos & ((1 << a.shift) - 1);
    const u16 *k = a.k + (c0 + i) * a.kt + h * a.kh + d, *v = a.v + (c0 + i) * a.vt + h * a.vh + d;
    u16 *ko = a.pk + p * a.kp + h * a.kph + t * a.kpt + d, *vo = a.pv + p * a.vp + h * a.vph + t * a.vpt + d;
    if constexpr (E == 8) {
        const uint4_t x0 = *gptr((const uint4_t*)k), x1 = *gptr((const uint4_t*)v);
        *gptr((uint4_t*)ko) = x0;
        *gptr((uint4_t*)vo) = x1;
    } else {
        *gptr(ko) = *gptr(k);
        *gptr(vo) = *gptr(v);
    }
}

constexpr int MAX_SEQS = 4096;         // of one table: a plan holds two words of LDS for each
int book_of(Book& a, int32_t* table, int32_t* lens, int32_t* refs, int32_t* free, int32_t* lack, int B, int per_seq, int pages, int page_rows) {
    if (!table || !lens || !refs || !free || !lack || B <= 0 || per_seq <= 0 || pages <= 0 || page_rows <= 0) return TCQ_ERR_ARG;
    if (B > MAX_SEQS || (int64_t)B * per_seq > 0x3fffffff || (int64_t)page_rows * per_seq > (1 << 30) || pages > (1 << 28)) return TCQ_ERR_UNSUPPORTED;
    if (((uintptr_t)table | (uintptr_t)lens | (uintptr_t)refs | (uintptr_t)free | (uintptr_t)lack) % 4) return TCQ_ERR_ALIGN;
    a = {table, lens, refs, (u32*)free, lack, B, per_seq, pages, (pages + 31) / 32, page_rows};
    return 0;
}
int copy_of(Copy& a, void* k, void* v, int layers, int pages, int64_t page_bytes) {
    if (!k || !v || layers <= 0 || pages <= 0 || page_bytes <= 0) return TCQ_ERR_ARG;
    if (page_bytes % 16 || ((uintptr_t)k | (uintptr_t)v) % 16) return TCQ_ERR_ALIGN;
    if (layers > 65536 || page_bytes > (1 << 28)) return TCQ_ERR_UNSUPPORTED;
    a = {};
    a.k = (char*)k, a.v = (char*)v, a.page = page_bytes, a.layer = page_bytes * pages, a.layers = layers, a.pages = pages;
    return 0;
}
int copy_run(const Copy& a, hipStream_t st) {
    const int64_t units = (a.page + CHUNK - 1) / CHUNK * a.layers * 2 * a.n;
    launch_k(k_pages_copy, dim3((u32)min(units, (int64_t)2048)), dim3(256), 0, st, a);
    return launch_status();
}

}  // namespace

extern "C" int tcq_pages_take(int32_t* table, int32_t* lens, int32_t* refs, int32_t* free, int32_t* lack, int B, int per_seq, int pages, int page_rows,
                              const int32_t* take, int32_t* start, void* k, void* v, int layers, int64_t page_bytes, int32_t* moves,
                              tcq_stream_t stream) {
    Book a;
    Copy c;
    int e = book_of(a, table, lens, refs, free, lack, B, per_seq, pages, page_rows);
    if (!e) e = copy_of(c, k, v, layers, pages, page_bytes);
    if (e) return e;
    if (!take || !start || !moves) return TCQ_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (B <= 256 && a.words <= 256) launch_k(k_pages_take<256>, dim3(1), dim3(256), (size_t)B * 8, st, a, take, start, moves);
    else launch_k(k_pages_take<1024>, dim3(1), dim3(1024), (size_t)B * 8, st, a, take, start, moves);
    if ((e = launch_status())) return e;
    c.count = moves, c.src = moves + 1, c.dst = moves + 1 + B, c.n = B;
    return copy_run(c, st);
}

extern "C" int tcq_pages_fork(int32_t* table, int32_t* lens, int32_t* refs, int32_t* free, int32_t* lack, int B, int per_seq, int pages, int page_rows,
                              const int32_t* src, const int32_t* dst, int n, tcq_stream_t stream) {
    Book a;
    const int e = book_of(a, table, lens, refs, free, lack, B, per_seq, pages, page_rows);
    if (e) return e;
    if (!src || !dst || n <= 0) return TCQ_ERR_ARG;
    if (n > 65535) return TCQ_ERR_UNSUPPORTED;
    launch_k(k_pages_fork, dim3(n), dim3(256), 0, (hipStream_t)stream, a, src, dst, n);
    return launch_status();
}

extern "C" int tcq_pages_trim(int32_t* table, int32_t* lens, int32_t* refs, int32_t* free, int32_t* lack, int B, int per_seq, int pages, int page_rows,
                              const int32_t* keep, tcq_stream_t stream) {
    Book a;
    const int e = book_of(a, table, lens, refs, free, lack, B, per_seq, pages, page_rows);
    if (e) return e;
    if (!keep) return TCQ_ERR_ARG;
    launch_k(k_pages_trim, dim3(B), dim3(64), 0, (hipStream_t)stream, a, keep);
    return launch_status();
}

extern "C" int tcq_pages_compact(int32_t* table, int32_t* lens, int32_t* refs, int32_t* free, int32_t* lack, int B, int per_seq, int pages,
                                 int page_rows, void* k, void* v, int layers, int64_t page_bytes, int32_t* moves, tcq_stream_t stream) {
    Book a;
    Copy c;
    int e = book_of(a, table, lens, refs, free, lack, B, per_seq, pages, page_rows);
    if (!e) e = copy_of(c, k, v, layers, pages, page_bytes);
    if (e) return e;
    if (!moves) return TCQ_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (a.words <= 256) launch_k(k_pages_plan<256>, dim3(1), dim3(256), 0, st, a, moves);
    else launch_k(k_pages_plan<1024>, dim3(1), dim3(1024), 0, st, a, moves);
    if ((e = launch_status())) return e;
    c.count = moves, c.from = moves + 1, c.src = moves + 2, c.dst = moves + 2 + pages / 2, c.to = moves + 2 + pages / 2 * 2, c.n = max(1, pages / 2);
    c.table = table, c.entries = B * per_seq;
    return copy_run(c, st);
}

extern "C" int tcq_pages_copy(void* k, void* v, int layers, int pages, int64_t page_bytes, const int32_t* src, const int32_t* dst, int n,
                              tcq_stream_t stream) {
    Copy c;
    const int e = copy_of(c, k, v, layers, pages, page_bytes);
    if (e) return e;
    if (!src || !dst || n <= 0) return TCQ_ERR_ARG;
    c.src = src, c.dst = dst, c.n = n;
    return copy_run(c, (hipStream_t)stream);
}

extern "C" int tcq_paged_append(const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, const int32_t* cu, int rows,
                                int most, int B, int H, int D, void* pk, int64_t k_page, int64_t pk_head, int64_t pk_tok, void* pv, int64_t v_page,
                                int64_t pv_head, int64_t pv_tok, int pages, int page_rows, const int32_t* table, int per_seq, const int32_t* lens,
                                const int32_t* start, tcq_stream_t stream) {
    if (!k || !v || !pk || !pv || !table || !lens || !start || rows <= 0 || most <= 0 || B <= 0 || H <= 0 || D <= 0 || pages <= 0 || per_seq <= 0)
        return TCQ_ERR_ARG;
    if (!cu && (int64_t)most * B > rows) return TCQ_ERR_SHAPE;
    if (page_rows < 16 || (page_rows & (page_rows - 1)) || page_rows > (1 << 20) || (int64_t)page_rows * per_seq > (1 << 30) || B > 65535 ||
        (int64_t)H * D > (1 << 24) || (int64_t)most * H * D / 256 > 0x7ffffff0)
        return TCQ_ERR_UNSUPPORTED;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)pk | (uintptr_t)pv) % 2 || ((uintptr_t)table | (uintptr_t)lens | (uintptr_t)start) % 4) return TCQ_ERR_ALIGN;
    const Append a = {(const u16*)k, (const u16*)v, k_tok, k_head, v_tok, v_head, (u16*)pk, (u16*)pv, k_page, pk_head, pk_tok, v_page, pv_head, pv_tok,
                      table, lens, start, cu, rows, most, H, D, per_seq, 31 - __builtin_clz(page_rows), pages};
    const bool vec = D % 8 == 0 && !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)pk | (uintptr_t)pv) % 16) &&
                     !((k_tok | k_head | v_tok | v_head | k_page | pk_head | pk_tok | v_page | pv_head | pv_tok) % 8);
    const int E = vec ? 8 : 1;
    const dim3 grid((u32)(((int64_t)most * (H * D / E) + 255) / 256), B);
    if (vec) launch_k(k_pages_append<8>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else launch_k(k_pages_append<1>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return launch_status();
}
