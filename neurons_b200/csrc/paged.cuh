// paged.cuh -- the paged key/value cache as its kernels see it, and the split
// of an attention call's work over the CTAs of a grid.
//
// A layer's cache is keys and values [n_pages][n_kv][page_size][head_dim]
// (pages page_stride elements apart).  Row s of the page table lists the pages
// of sequence s and lens[s] is its length, new tokens included.  The batch
// names its sequences by table row; the new tokens of entry b are rows
// q_starts[b] .. q_starts[b + 1] of q and stand at the sequence's end.
#pragma once

#include <cuda.h>

#include <atomic>

#include "nq_common.cuh"

namespace nq {

struct PagedBatch {
    const int32_t *table;     // [n_rows][table_ld], table_width entries each; -1: no page
    const int32_t *lens;      // [n_rows]
    const int32_t *seqs;      // [n_seqs] table row of entry b (< 0: padding); nullptr: b
    const int32_t *q_starts;  // [n_seqs + 1]; nullptr: entry b is row b of q
    int64_t table_ld;
    int table_width, n_rows, n_seqs, n_tokens;
    int page_size, n_pages;
    unsigned *err;
};

// One entry of the batch: table row, first row of q, new tokens, length.
struct SeqView {
    int row, q0, n, len;
};

// Reads entry b.  What the arrays say outside their ranges (a table row, a
// length past the table's width, token rows past n_tokens) is cut to the range
// and raises the error word, and is told in *cut; a padding entry has n == 0.
// (All loads first: each is a trip to L2, and a call waits for them before its
// first key.)
__device__ __forceinline__ SeqView seq_view(const PagedBatch &pb, int b, bool *cut = nullptr) {
    SeqView s;
    s.row = pb.seqs ? pb.seqs[b] : b;
    int end = b + 1;
    s.q0 = b;
    if (pb.q_starts) {
        s.q0 = pb.q_starts[b];
        end = pb.q_starts[b + 1];
    }
    s.len = pb.lens[min(max(s.row, 0), pb.n_rows - 1)];
    s.n = end - s.q0;
    bool bad = false;
    if (s.q0 < 0 || s.q0 > pb.n_tokens || end < s.q0) {
        bad = true;
        s.q0 = 0;
        s.n = 0;
    } else if (end > pb.n_tokens) {
        bad = true;
        s.n = pb.n_tokens - s.q0;
    }
    const int64_t most = (int64_t)pb.table_width * pb.page_size;
    if (s.row < 0) {
        s.n = 0;
        s.len = 0;
    } else if (s.row >= pb.n_rows) {
        bad = true;
        s.row = 0;
        s.len = 0;
    } else if (s.len < 0 || s.len > most) {
        bad = true;
        s.len = s.len < 0 ? 0 : (int)most;
    }
    if (bad) atomicOr(pb.err, kErrBadIndex);
    if (cut) *cut = bad;
    return s;
}

// Key blocks [lo, lo + nb) of `BK` keys that the new tokens [t0, t1) of a
// sequence see (position of token t: len - n + t; keys up to it, and within
// the window when there is one).  nb is at least 1, so that rows without any
// key have a block, all of it masked, that writes their zeros.
struct KeyRange {
    int lo, nb;
};

template <int BK>
__device__ __forceinline__ KeyRange key_range(const SeqView &s, int t0, int t1, int window) {
    const int p0 = s.len - s.n + t0, p1 = s.len - s.n + t1 - 1;
    KeyRange r;
    const int hi = p1 < 0 ? 0 : p1 / BK + 1;
    r.lo = window > 0 && p0 - window + 1 > 0 ? (p0 - window + 1) / BK : 0;
    r.nb = hi - r.lo;
    if (r.nb < 1) {
        r.lo = max(0, hi - 1);
        r.nb = 1;
    }
    return r;
}

// How a kernel cuts an entry's new tokens: tiles of TT tokens.  A key block costs
// 3 units of work for a tile of up to `half` tokens and 4 for a larger one
// (attn_paged_tc.cu, 1.6 and 2.2 us at 128 dims).
struct Tiling {
    static constexpr int kMost = 4;
    int TT, half, window;
    bool whole;  // a tile counts as one unit and is never cut
    __device__ __forceinline__ int tiles(int n) const { return n <= TT ? n > 0 : (n + TT - 1) / TT; }
    __device__ __forceinline__ int weight(int t0, int t1) const { return t1 - t0 > half ? 4 : 3; }
};

// A position in the list of all units of a call: entry b, key head h, place t in
// the order of the token tiles, and `off` units into that tile; `at` is its
// number and `left` what the CTA still has to do; done: it stands at the end of
// tile t.  (The step to the next tile is taken with the next piece: it may wait
// for memory, which a piece in hand need not.)
struct Cursor {
    int b, h, t, off;
    bool done;
    int64_t at, left;
    SeqView s;
};

// The token tile at place i of n: first, last, second, last but one, ...  A
// prompt's first tiles see few keys and its last ones many; in this order each
// stretch of the list holds both, and no CTA gets only short tiles, whose
// beginnings and ends cost more than their products.
__device__ __forceinline__ int tile_at(int i, int n) { return i & 1 ? n - 1 - (i >> 1) : i >> 1; }

// Units of the tile at place i of `tiles`.
template <int BK>
__device__ __forceinline__ int tile_units(const SeqView &s, const Tiling &tl, int i, int tiles) {
    const int t0 = tile_at(i, tiles) * tl.TT, t1 = min(t0 + tl.TT, s.n);
    return key_range<BK>(s, t0, t1, tl.window).nb * tl.weight(t0, t1);
}

// The list: entries in order, in each its key heads, in each the token tiles in
// tile_at()'s order, in each its key blocks.  Neighbouring CTAs therefore read
// the same head's keys at the same time.  CTA c of n takes the units
// [c * total / n, (c + 1) * total / n) (a block goes with its first unit), so
// that all CTAs get the same work whatever the lengths are; a tile cut by such a
// border is finished by a merge kernel.  Where no sequence can be long (`whole`)
// a tile counts as one and is never cut: no parts, and no merge.
template <int BK>
__device__ __forceinline__ int64_t entry_units_warp(const SeqView &s, const Tiling &tl) {
    // units of one head of this lane's entry; the lanes sum long entries together
    const int lane = threadIdx.x & 31;
    const int tiles = tl.tiles(s.n);
    if (tl.whole) return tiles;
    int64_t mine = 0;
    if (tiles == 1) mine = tile_units<BK>(s, tl, 0, 1);
    unsigned todo = __ballot_sync(0xffffffffu, tiles > 1);
    while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        SeqView o;
        o.n = __shfl_sync(0xffffffffu, s.n, src);
        o.len = __shfl_sync(0xffffffffu, s.len, src);
        const int ot = tl.tiles(o.n);
        int64_t sum = 0;
        for (int t = lane; t < ot; t += 32) sum += tile_units<BK>(o, tl, t, ot);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == src) mine = sum;
    }
    return mine;
}

// Sums over the warp's lanes of values >= 0; in 32 bits where they fit, which is
// less of the chain that a call's first key waits for.
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
    if (!__any_sync(0xffffffffu, v >> 26)) return __reduce_add_sync(0xffffffffu, (unsigned)v);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ int64_t warp_inclusive(int64_t v) {
    const int lane = threadIdx.x & 31;
    if (!__any_sync(0xffffffffu, v >> 26)) {
        int x = (int)v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += o;
        }
        return x;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// What a CTA does.
struct Share {
    int64_t total;   // units of the call
    int n;           // CTAs that take part
    Cursor c;        // at this CTA's first unit; c.left of them
};

// a * b / c; in 32 bits, which is several times faster, where the product fits
__device__ __forceinline__ int64_t mul_div(int64_t a, int64_t b, int64_t c) {
    if (((a | b | c) >> 32) == 0 && a * b < (1ll << 32))
        return (uint32_t)(a * b) / (uint32_t)c;
    return a * b / c;
}

// CTAs that take part in a call of `total` units: no share is smaller than a
// block's units (every share between a tile's first and last one then holds a
// block of it), or a whole tile.
__device__ __forceinline__ int sharers(int64_t total, int grid, bool whole) {
    const int least = whole ? 1 : Tiling::kMost;
    if (total >= (int64_t)grid * least) return grid;
    const int n = whole ? (int)total : (int)total / Tiling::kMost;
    return n > 0 ? n : 1;
}
__device__ __forceinline__ int64_t share_start(int64_t total, int n, int c) {
    return mul_div(c, total, n);
}
// the CTA whose share holds unit u
__device__ __forceinline__ int share_owner(int64_t total, int n, int64_t u) {
    if ((u + 1) * n - 1 < (1ll << 32) && total < (1ll << 32))
        return (int)((uint32_t)((u + 1) * n - 1) / (uint32_t)total);
    return (int)(((u + 1) * n - 1) / total);
}

// Run by one whole warp.
template <int BK>
__device__ __forceinline__ Share find_share(const PagedBatch &pb, int n_kv, const Tiling &tl,
                                            int cta, int grid) {
    const int lane = threadIdx.x & 31;
    Share sh;
    SeqView s{0, 0, 0, 0};
    int64_t head = 0, total = 0;
    for (int b0 = 0; b0 < pb.n_seqs; b0 += 32) {
        s = SeqView{0, 0, 0, 0};
        if (b0 + lane < pb.n_seqs) s = seq_view(pb, b0 + lane);
        head = entry_units_warp<BK>(s, tl);
        total += head;
    }
    sh.total = warp_sum(total) * n_kv;
    sh.n = sharers(sh.total, grid, tl.whole);
    sh.c = Cursor{0, 0, 0, 0, false, 0, 0, SeqView{0, 0, 0, 0}};
    if (sh.total == 0 || cta >= sh.n) return sh;
    Cursor &c = sh.c;
    c.at = share_start(sh.total, sh.n, cta);
    c.left = share_start(sh.total, sh.n, cta + 1) - c.at;
    int64_t before = 0;
    for (int b0 = 0; b0 < pb.n_seqs; b0 += 32) {
        if (pb.n_seqs > 32) {  // (else the first pass left them)
            s = SeqView{0, 0, 0, 0};
            if (b0 + lane < pb.n_seqs) s = seq_view(pb, b0 + lane);
            head = entry_units_warp<BK>(s, tl);
        }
        const int64_t end = before + warp_inclusive(head * n_kv);
        const unsigned past = __ballot_sync(0xffffffffu, end > c.at);
        if (past) {
            const int src = __ffs(past) - 1;
            c.b = b0 + src;
            c.s.row = __shfl_sync(0xffffffffu, s.row, src);
            c.s.q0 = __shfl_sync(0xffffffffu, s.q0, src);
            c.s.n = __shfl_sync(0xffffffffu, s.n, src);
            c.s.len = __shfl_sync(0xffffffffu, s.len, src);
            const int64_t per = __shfl_sync(0xffffffffu, head, src);
            int64_t at = c.at - (__shfl_sync(0xffffffffu, end, src) - per * n_kv);
            c.h = (int)mul_div(at, 1, per);
            at -= c.h * per;
            const int tiles = tl.tiles(c.s.n);
            if (tiles == 1) {
                c.off = (int)at;
                return sh;
            }
            int64_t seen = 0;
            for (int i0 = 0; i0 < tiles; i0 += 32) {
                int64_t u = 0;
                if (i0 + lane < tiles)
                    u = tl.whole ? 1 : tile_units<BK>(c.s, tl, i0 + lane, tiles);
                const int64_t e = seen + warp_inclusive(u);
                const unsigned over = __ballot_sync(0xffffffffu, e > at);
                if (over) {
                    const int l = __ffs(over) - 1;
                    c.t = i0 + l;
                    c.off = (int)(at - __shfl_sync(0xffffffffu, e - u, l));
                    break;
                }
                seen = __shfl_sync(0xffffffffu, e, 31);
            }
            return sh;
        }
        before = __shfl_sync(0xffffffffu, end, 31);
    }
    return sh;
}

// One piece of work: blocks [k0, k1) of the nb blocks of a tile, which begin
// at key block lo.
struct Piece {
    SeqView s;
    int h, t0, t1;     // key head; new tokens [t0, t1)
    int lo, k0, k1, nb;
    int parts;         // of a tile that this piece begins and does not finish; else 0
};

// Takes the next piece of a share and steps past it; false when done.  (Any
// thread: no warp-wide step.)
template <int BK>
__device__ __forceinline__ bool next_piece(const PagedBatch &pb, int n_kv, const Tiling &tl,
                                           Share &sh, int cta, Piece &p) {
    Cursor &c = sh.c;
    while (c.left > 0) {
        if (c.done) {
            c.done = false;
            c.off = 0;
            if (++c.t == tl.tiles(c.s.n)) {
                c.t = 0;
                if (++c.h == n_kv) {
                    c.h = 0;
                    do {
                        c.s = seq_view(pb, ++c.b);
                    } while (c.s.n == 0);
                }
            }
        }
        p.s = c.s;
        p.h = c.h;
        const int tiles = tl.tiles(c.s.n);
        p.t0 = tile_at(c.t, tiles) * tl.TT;
        p.t1 = min(p.t0 + tl.TT, c.s.n);
        const KeyRange r = key_range<BK>(c.s, p.t0, p.t1, tl.window);
        p.lo = r.lo;
        p.nb = r.nb;
        p.k0 = 0;
        p.k1 = r.nb;
        p.parts = 0;
        int end = 1, off = 1;  // the tile's units, and those before the next piece
        if (!tl.whole) {
            const int w = tl.weight(p.t0, p.t1);
            end = r.nb * w;
            off = (int)min((int64_t)end, c.off + c.left);
            auto blocks = [&](int units) { return w == 4 ? (units + 3) / 4 : (units + 2) / 3; };
            p.k0 = blocks(c.off);
            p.k1 = blocks(off);
            if (p.k0 == 0 && p.k1 < r.nb)
                p.parts = share_owner(sh.total, sh.n, c.at - c.off + end - w) - cta + 1;
        }
        const int took = off - c.off;
        c.left -= took;
        c.at += took;
        c.off = off;
        c.done = off == end;
        if (p.k0 < p.k1) return true;
    }
    return false;
}

// page of key `key` of table row `row`; n_pages (whose reads give zeros) when
// the table holds none there, which raises the error word
__device__ __forceinline__ int page_of(const PagedBatch &pb, int row, int key) {
    const int p = pb.table[(int64_t)row * pb.table_ld + key / pb.page_size];
    if (p >= 0 && p < pb.n_pages) return p;
    atomicOr(pb.err, kErrBadIndex);
    return pb.n_pages;
}

// A tile whose blocks several CTAs share: CTA c's part goes to slot 2c + 1 when
// it begins the tile, else 2c; the CTA that begins a tile it does not finish
// leaves this note for the merge (parts == 0: none).
struct SplitNote {
    int q_row, heads0, tokens, parts;
};

// Whether the merge may follow CTA `cta`'s note: its parts and rows lie within
// the call.  A call's own notes do; those that an overlapping call left in a
// workspace used twice need not, and they say where the merge reads and writes.
__host__ __device__ __forceinline__ bool note_fits(const SplitNote &n, int cta, int ctas, int n_tokens,
                                                   int n_heads, int group) {
    return n.parts > 0 && n.parts <= ctas - cta && n.q_row >= 0 && n.tokens > 0 &&
           n.tokens <= n_tokens && n.q_row <= n_tokens - n.tokens && n.heads0 >= 0 &&
           n.heads0 <= n_heads - group;
}

// mbar_wait_or_abort() by a whole warp, which goes on or gives up as one: where its
// lanes could part, those that go on would wait in the next warp-wide step for
// those that have left.
__device__ __forceinline__ bool warp_wait_or_abort(uint64_t *bar, uint32_t parity,
                                                   volatile int *abort, unsigned *err) {
    return __all_sync(0xffffffffu, mbar_wait_or_abort(bar, parity, abort, err)) != 0;
}

// An attention call as its kernels take it.
struct PagedAttnArgs {
    PagedBatch pb;
    const uint16_t *q;   // [n_tokens][q_ld]: n_heads x head_dim each
    uint16_t *out;       // [n_tokens][out_ld]
    int64_t q_ld, out_ld;
    int n_heads, n_kv, window;
    int box, box_cols;   // keys and columns of 64 dims per TMA box
    bool whole;          // tiles are not cut
    float scale;
    SplitNote *notes;    // [CTAs]
    float *part_ml;      // [2 CTAs][rows][2]: maximum (times scale log2 e), sum
    float *part_o;       // [2 CTAs][rows][head_dim]
};

// A checked call, as the C ABI hands it to launch_paged_attention.
struct PagedAttnCall {
    PagedBatch pb;
    const uint16_t *q, *k, *v;
    uint16_t *out;
    int64_t q_ld, out_ld, page_stride, max_q;
    int n_heads, n_kv, head_dim, window;
    bool f16;
    float scale;
    void *ws;
};

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// max_keys: the longest sequence that the page table can hold
size_t paged_attention_workspace(int n_heads, int n_kv, int head_dim, int64_t max_q,
                                 int64_t max_keys);
cudaError_t launch_paged_attention(const PagedAttnCall &c, cudaStream_t st);

// attn_paged_tc.cu: rows of its parts, and its launch (one CTA per SM)
int paged_tiles_rows(int head_dim);
cudaError_t launch_paged_tiles(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                               int hd, bool f16, cudaStream_t st);

// Allows a kernel `bytes` of dynamic shared memory, once per device (`done`: a
// bit per device, one word for each kernel).
template <typename K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t> &done) {
    int d = 0;
    cudaError_t e = cudaGetDevice(&d);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (d & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem,
                       cudaStream_t stream, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

__device__ __forceinline__ void tma_load_4d(void *smem_dst, const void *tmap, uint64_t *bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void tma_load_5d(void *smem_dst, const void *tmap, uint64_t *bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3,
                                            int32_t c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

}  // namespace nq
