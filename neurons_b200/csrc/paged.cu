// paged.cu -- the paged key/value cache around its attention (attn_paged.cu):
// the append of new tokens with their rotary positions, the page pool's fork,
// reserve, free, compact and copy, and the C ABI of all of them.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "nq.h"
#include "nq_common.cuh"
#include "nq_internal.h"
#include "paged.cuh"

namespace nq {
namespace {

// ------------------------------------------------------------------- append

struct AppendArgs {
    PagedBatch pb;
    const uint16_t *q, *k, *v;  // rows of n_heads / n_kv / n_kv heads, ld elements apart
    uint16_t *q_out, *kc, *vc;
    const float *freqs;         // [half] radians per position
    int64_t q_ld, k_ld, v_ld, q_out_ld, page_stride;
    int n_heads, n_kv, hd, half;
};

// The entry of the batch that holds token i: the last one that starts at or
// before it.  Run by a whole warp; 32 starts per step.
__device__ __forceinline__ int entry_of(const PagedBatch &pb, int i) {
    if (!pb.q_starts) return i < pb.n_seqs ? i : -1;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = pb.n_seqs;  // the entry is in [lo, lo + n)
    while (n > 0) {
        const int step = (n + 31) / 32;
        const int b = lo + lane * step;
        const bool in = lane * step < n && pb.q_starts[b] <= i;
        const int c = __popc(__ballot_sync(0xffffffffu, in));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (step == 1) return lo;
    }
    return -1;
}

constexpr int kAppendThreads = 128;

// (x_i, x_{i + half}) turned by pos * freqs[i], for the first 2 * half dims of
// each head of q and k; the rest, and v, as they are.  k and v go to their
// page.  One CTA per token: its angles are computed once for all heads.
// Memory bounds it: the first three vector pairs and one value vector of a thread
// (all there are for 40 turned heads of 128 dims) are under way before the token's
// entry, page and angles are looked up (four chunks of 11091 tokens 69 -> 49 us
// when it came; 51 to 54 us over several GPUs, 5.1 to 5.3 TB/s).
template <bool F16>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float2 turn[128];  // cosine, sine
    const int64_t i = blockIdx.x;
    const int tid = threadIdx.x;
    const int per = a.half / 8, heads = a.n_heads + a.n_kv, pairs = heads * per;
    const int vper = a.hd / 8, values = a.n_kv * vper;
    // vector pair w of the token: its first half (the second is a.half on)
    auto source = [&](int w) {
        const int h = w / per, f = (w - h * per) * 8;
        return (h < a.n_heads ? a.q + i * a.q_ld + (int64_t)h * a.hd
                              : a.k + i * a.k_ld + (int64_t)(h - a.n_heads) * a.hd) +
               f;
    };
    auto value = [&](int w) {
        const int h = w / vper;
        return a.v + i * a.v_ld + (int64_t)h * a.hd + (w - h * vper) * 8;
    };
    constexpr int kFirst = 3;
    uint4 x[kFirst], y[kFirst], vv = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kFirst; ++j) {
        const int w = tid + j * kAppendThreads;
        if (w < pairs) {
            const uint16_t *src = source(w);
            x[j] = *reinterpret_cast<const uint4 *>(src);
            y[j] = *reinterpret_cast<const uint4 *>(src + a.half);
        }
    }
    if (tid < values) vv = *reinterpret_cast<const uint4 *>(value(tid));

    const int b = entry_of(a.pb, (int)i);
    if (b < 0) return;
    bool cut;
    const SeqView s = seq_view(a.pb, b, &cut);
    // (counted from a cut length the tokens would be written over the keys before them)
    if (cut) return;
    const int t = (int)i - s.q0;
    if (t < 0 || t >= s.n) return;  // behind the last sequence, or padding
    const int pos = s.len - s.n + t;
    for (int f = tid; f < a.half; f += kAppendThreads) turn[f] = rope_turn(pos, a.freqs[f]);
    int page = a.pb.n_pages;
    if (pos >= 0)
        page = page_of(a.pb, s.row, pos);
    else if (tid == 0)
        atomicOr(a.pb.err, kErrBadIndex);  // more new tokens than the length
    __syncthreads();
    const int64_t place =
        (int64_t)page * a.page_stride + (int64_t)(pos < 0 ? 0 : pos % a.pb.page_size) * a.hd;
    const int64_t head_ld = (int64_t)a.pb.page_size * a.hd;  // next key head's row in a page
    const bool keep = page < a.pb.n_pages;
    // where head h of q and k goes (nullptr: nowhere)
    auto target = [&](int h) -> uint16_t * {
        if (h < a.n_heads) return a.q_out + i * a.q_out_ld + (int64_t)h * a.hd;
        return keep ? a.kc + place + (h - a.n_heads) * head_ld : nullptr;
    };
    auto put_pair = [&](int w, const uint4 &xv, const uint4 &yv) {
        const int h = w / per, f = (w - h * per) * 8;
        const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w}, ys[4] = {yv.x, yv.y, yv.z, yv.w};
        uint32_t u[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float p[2], r[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 cs = turn[f + 2 * j + e];
                const float x1 = t16_to_f32<F16>((uint16_t)(xs[j] >> (16 * e)));
                const float x2 = t16_to_f32<F16>((uint16_t)(ys[j] >> (16 * e)));
                p[e] = x1 * cs.x - x2 * cs.y;
                r[e] = x1 * cs.y + x2 * cs.x;
            }
            u[j] = pack_t2<F16>(p[0], p[1]);
            v[j] = pack_t2<F16>(r[0], r[1]);
        }
        uint16_t *dst = target(h);
        if (!dst) return;
        *reinterpret_cast<uint4 *>(dst + f) = make_uint4(u[0], u[1], u[2], u[3]);
        *reinterpret_cast<uint4 *>(dst + f + a.half) = make_uint4(v[0], v[1], v[2], v[3]);
    };
    auto put_value = [&](int w, const uint4 &v) {
        const int h = w / vper;
        if (keep)
            *reinterpret_cast<uint4 *>(a.vc + place + h * head_ld + (w - h * vper) * 8) = v;
    };
#pragma unroll
    for (int j = 0; j < kFirst; ++j) {
        const int w = tid + j * kAppendThreads;
        if (w < pairs) put_pair(w, x[j], y[j]);
    }
    if (tid < values) put_value(tid, vv);
    for (int w = tid + kFirst * kAppendThreads; w < pairs; w += kAppendThreads) {
        const uint16_t *src = source(w);
        put_pair(w, *reinterpret_cast<const uint4 *>(src),
                 *reinterpret_cast<const uint4 *>(src + a.half));
    }
    for (int w = tid + kAppendThreads; w < values; w += kAppendThreads)
        put_value(w, *reinterpret_cast<const uint4 *>(value(w)));
    const int rest = (a.hd - 2 * a.half) / 8;  // vectors of a head that are not turned
    for (int w = tid; w < heads * rest; w += kAppendThreads) {
        const int h = w / rest, f = 2 * a.half + (w - h * rest) * 8;
        const uint16_t *src = h < a.n_heads ? a.q + i * a.q_ld + (int64_t)h * a.hd
                                            : a.k + i * a.k_ld + (int64_t)(h - a.n_heads) * a.hd;
        if (uint16_t *dst = target(h))
            *reinterpret_cast<uint4 *>(dst + f) = *reinterpret_cast<const uint4 *>(src + f);
    }
}

// ---------------------------------------------------------------- page pool

struct PageTable {
    int32_t *refs;   // [n_pages] sequences that hold the page
    int32_t *table;  // [n_rows][table_ld]
    int32_t *lens;   // [n_rows]
    int64_t table_ld;
    int table_width, n_rows, n_pages, page_size;
    unsigned *err;
};

// whether x is among list[0, n); by the whole block
__device__ __forceinline__ bool block_has(const int32_t *list, int n, int x) {
    int hit = 0;
    for (int j = threadIdx.x; j < n; j += blockDim.x) hit |= list[j] == x;
    return __syncthreads_or(hit) != 0;
}

// One CTA per listed sequence: its pages lose a holder.  The second and later
// mentions of a sequence find nothing to do.
__global__ void __launch_bounds__(256) pages_free_kernel(const PageTable a, const int32_t *seqs) {
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x, s = seqs[i];
    if (s < 0) return;  // padding
    if (s >= a.n_rows) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrPages);
        return;
    }
    if (block_has(seqs, i, s)) return;
    int32_t *row = a.table + s * a.table_ld;
    for (int j = threadIdx.x; j < a.table_width; j += blockDim.x) {
        const int p = row[j];
        if (p == -1) continue;
        if (p >= 0 && p < a.n_pages)
            atomicSub(&a.refs[p], 1);
        else
            atomicOr(a.err, kErrPages);
        row[j] = -1;
    }
    if (threadIdx.x == 0) a.lens[s] = 0;
}

// One CTA per pair: the child gets its parent's pages, each with a holder
// more.  Refused (error word, the pair does nothing): rows out of range, a
// child that has tokens or pages, is listed before, or is a parent in this
// call.
__global__ void __launch_bounds__(256) pages_fork_kernel(const PageTable a, const int32_t *parents,
                                                         const int32_t *children, int n) {
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x, p = parents[i], c = children[i];
    if (p < 0 && c < 0) return;  // padding
    bool bad = p < 0 || p >= a.n_rows || c < 0 || c >= a.n_rows;
    if (!bad) {
        bad = block_has(children, i, c);
        bad |= block_has(parents, n, c);
        bad |= block_has(children, n, p);
    }
    // a child is read only when no other pair writes it
    if (!bad) bad = a.lens[c] != 0 || a.table[c * a.table_ld] != -1;
    if (bad) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrPages);
        return;
    }
    __syncthreads();  // every thread has read the child's state
    const int32_t *src = a.table + p * a.table_ld;
    int32_t *dst = a.table + c * a.table_ld;
    for (int j = threadIdx.x; j < a.table_width; j += blockDim.x) {
        const int page = src[j];
        dst[j] = page;
        if (page >= 0 && page < a.n_pages) atomicAdd(&a.refs[page], 1);
    }
    if (threadIdx.x == 0) a.lens[c] = a.lens[p];
}

constexpr int kPlanThreads = 1024;

// exclusive sum over the block of v; *total gets the whole sum
__device__ __forceinline__ int block_exclusive(int v, int *total) {
    __shared__ int sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += o;
    }
    __syncthreads();  // (the last call's sums have been read)
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int y = sums[lane], z = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, z, d);
        if (lane >= d) z += o;
    }
    *total = __shfl_sync(0xffffffffu, z, 31);
    const int before = __shfl_sync(0xffffffffu, z - y, warp);
    return before + x - v;
}

// Page moves that a copy kernel makes: count, then (from, to) pairs.
struct Moves {
    int32_t *count;
    int2 *pair;
};

// Every listed sequence grows to its new length, in the list's order: a last
// page that is not full and has other holders is replaced by a free one (its
// contents follow in the copy kernel), then free pages are added, always the
// lowest.  Of several listed holders of one page all but the last get copies
// when nobody else holds it.  All or nothing: a length below the present one
// or past the table's width, a sequence listed twice, a row out of range or
// too few free pages raise the error word and leave everything as it was.
// One CTA; the per-entry state is in `ws` ([3][n] int32).
__global__ void __launch_bounds__(kPlanThreads) pages_reserve_kernel(
    const PageTable a, const int32_t *seqs, const int32_t *new_lens, int n, int32_t *ws, Moves mv) {
    pdl_launch_dependents();
    pdl_wait();
    int32_t *last = ws, *first = ws + n, *offset = ws + 2 * n;  // offset: of its first new page
    const int tid = threadIdx.x;
    int bad = 0, shared_pages = 0;
    for (int i = tid; i < n; i += kPlanThreads) {
        const int s = seqs[i];
        int lp = -1;
        if (s >= 0) {
            const int old = s < a.n_rows ? a.lens[s] : -1, now = new_lens[i];
            if (old < 0 || now < old || now > (int64_t)a.table_width * a.page_size) {
                bad = 1;
            } else if (now > old && old % a.page_size) {
                const int page = a.table[s * a.table_ld + old / a.page_size];
                if (page < 0 || page >= a.n_pages)
                    bad = 1;
                else if (a.refs[page] > 1)
                    lp = page;
            }
        }
        last[i] = lp;
        shared_pages |= lp >= 0;
    }
    shared_pages = __syncthreads_or(shared_pages);
    for (int i = tid; i < n; i += kPlanThreads) {  // listed twice?
        const int s = seqs[i];
        if (s >= 0)
            for (int j = 0; j < i; ++j) bad |= seqs[j] == s;
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) {
            atomicOr(a.err, kErrPages);
            *mv.count = 0;
        }
        return;
    }
    // who copies: every holder but the last of those that hold the page alone
    int total = 0, copies = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int need = 0, split = 0;
        if (i < n && seqs[i] >= 0) {
            const int s = seqs[i], old = a.lens[s], now = new_lens[i];
            if (shared_pages && last[i] >= 0) {
                int rank = 0;
                for (int j = 0; j < i; ++j) rank += last[j] == last[i];
                split = rank < a.refs[last[i]] - 1;
            }
            const int have = (old + a.page_size - 1) / a.page_size;
            first[i] = have - split;
            need = max(0, (now + a.page_size - 1) / a.page_size - have) + split;
        }
        int sum;
        const int at = block_exclusive(need, &sum);
        if (i < n) offset[i] = total + at;
        total += sum;
        const int ca = block_exclusive(split, &sum);
        // (the pair's target page follows below; x marks the entry)
        if (split) mv.pair[copies + ca] = make_int2(last[i], -1 - i);
        copies += sum;
    }
    // are there enough free pages?
    int seen = 0;
    for (int p0 = 0; p0 < a.n_pages && seen < total; p0 += kPlanThreads) {
        const int p = p0 + tid;
        int sum = __syncthreads_count(p < a.n_pages && a.refs[p] == 0);
        seen += sum;
    }
    if (seen < total) {
        if (tid == 0) {
            atomicOr(a.err, kErrPages);
            *mv.count = 0;
        }
        return;
    }
    // hand them out: the k-th free page goes to the entry whose range holds k
    seen = 0;
    for (int p0 = 0; seen < total; p0 += kPlanThreads) {
        const int p = p0 + tid;
        const int is_free = p < a.n_pages && a.refs[p] == 0;
        int sum;
        const int k = seen + block_exclusive(is_free, &sum);
        if (is_free && k < total) {
            int lo = 0, hi = n;  // the last entry with offset <= k that takes pages
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (offset[mid] <= k)
                    lo = mid;
                else
                    hi = mid;
            }
            a.table[seqs[lo] * a.table_ld + first[lo] + k - offset[lo]] = p;
            a.refs[p] = 1;
        }
        seen += sum;
    }
    __syncthreads();
    for (int m = tid; m < copies; m += kPlanThreads) {
        const int2 x = mv.pair[m];
        const int i = -1 - x.y;
        mv.pair[m].y = a.table[seqs[i] * a.table_ld + first[i]];
        atomicSub(&a.refs[x.x], 1);
    }
    for (int i = tid; i < n; i += kPlanThreads)
        if (seqs[i] >= 0) a.lens[seqs[i]] = new_lens[i];
    if (tid == 0) *mv.count = copies;
}

// The used pages past the number of used pages move to the free ones below it,
// lowest to lowest.  One CTA; `to` [n_pages] gets the moved pages' new places.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_kernel(const PageTable a, int32_t *to,
                                                                     Moves mv) {
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x;
    int used = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += kPlanThreads)
        used += __syncthreads_count(p0 + tid < a.n_pages && a.refs[p0 + tid] != 0);
    int holes = 0, moved = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += kPlanThreads) {
        const int p = p0 + tid;
        const bool in = p < a.n_pages, held = in && a.refs[p] != 0;
        const int hole = in && p < used && !held, move = held && p >= used;
        if (in && p >= used) to[p] = p;  // (an entry without a holder stays)
        int sum;
        const int h = block_exclusive(hole, &sum);
        if (hole) mv.pair[holes + h].y = p;
        holes += sum;
        const int m = block_exclusive(move, &sum);
        if (move) mv.pair[moved + m].x = p;
        moved += sum;
    }
    __syncthreads();
    for (int m = tid; m < moved; m += kPlanThreads) {
        const int2 x = mv.pair[m];
        to[x.x] = x.y;
        a.refs[x.y] = a.refs[x.x];
        a.refs[x.x] = 0;
    }
    if (tid == 0) {
        mv.count[0] = moved;
        mv.count[1] = used;
    }
}

struct PagePool {
    uint8_t *data;  // [outer][n_pages][page_bytes]
    int64_t outer, page_bytes;
    int n_pages;
};

// Four 16-byte vectors a thread and step: 2.85 GB of reads and writes take 476 us,
// 0.92 of a plain copy's rate; eight vectors, or loads that pass by the caches,
// gained nothing.
constexpr int kCopyThreads = 256, kCopyBytes = kCopyThreads * 16 * 4;  // per step of a CTA

__device__ __forceinline__ void copy_piece(const PagePool &pool, int from, int to, int64_t o,
                                           int64_t at) {
    const uint8_t *src = pool.data + (o * pool.n_pages + from) * pool.page_bytes;
    uint8_t *dst = pool.data + (o * pool.n_pages + to) * pool.page_bytes;
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t b = at + (j * kCopyThreads + threadIdx.x) * 16;
        if (b < pool.page_bytes) v[j] = *reinterpret_cast<const uint4 *>(src + b);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t b = at + (j * kCopyThreads + threadIdx.x) * 16;
        if (b < pool.page_bytes) *reinterpret_cast<uint4 *>(dst + b) = v[j];
    }
}

// The moves' pages, all layers; `to` (compaction): also the table's entries.
__global__ void __launch_bounds__(kCopyThreads) pages_move_kernel(const PagePool pool,
                                                                  const Moves mv, const PageTable a,
                                                                  const int32_t *to) {
    pdl_launch_dependents();
    pdl_wait();
    const int count = mv.count[0];
    const int64_t pieces = (pool.page_bytes + kCopyBytes - 1) / kCopyBytes;
    const int64_t per = pool.outer * pieces, n = count * per;
    for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
        const int2 x = mv.pair[w / per];
        const int64_t r = w % per;
        copy_piece(pool, x.x, x.y, r / pieces, r % pieces * kCopyBytes);
    }
    if (to && count > 0) {
        const int used = mv.count[1];
        const int64_t cells = (int64_t)a.n_rows * a.table_width;
        for (int64_t w = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; w < cells;
             w += (int64_t)gridDim.x * kCopyThreads) {
            int32_t *e = a.table + w / a.table_width * a.table_ld + w % a.table_width;
            if (*e >= used && *e < a.n_pages) *e = to[*e];
        }
    }
}

// The caller's own moves.  A move whose target is another move's source, or a
// target listed before, would race: it is not made and raises the error word.
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const PagePool pool,
                                                                  const int32_t *src,
                                                                  const int32_t *dst, int n,
                                                                  unsigned *err) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t pieces = (pool.page_bytes + kCopyBytes - 1) / kCopyBytes;
    const int64_t per = pool.outer * pieces;
    for (int m = blockIdx.x; m < n; m += gridDim.x) {
        const int from = src[m], to = dst[m];
        if ((from < 0 && to < 0) || from == to) continue;  // padding, or in place
        bool bad = from < 0 || from >= pool.n_pages || to < 0 || to >= pool.n_pages;
        if (!bad) {
            bad = block_has(dst, m, to);
            bad |= block_has(src, n, to);
        }
        if (bad) {
            if (threadIdx.x == 0) atomicOr(err, kErrPages);
            continue;
        }
        for (int64_t r = blockIdx.y; r < per; r += gridDim.y)
            copy_piece(pool, from, to, r / pieces, r % pieces * kCopyBytes);
    }
}

int fail(int status, const std::string &msg) {
    set_error(msg);
    return status;
}

int from_cuda(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return NQ_SUCCESS;
    cudaGetLastError();
    return fail(NQ_COMPUTE_ERROR, std::string(what) + ": " + cudaGetErrorString(e));
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int64_t kMaxInt = 0x7fffffff;

// The longest lists that are taken.  The kernels compare each entry with those
// before it, so their time grows with the square of the length: 65536 entries
// take the reserve's one CTA 49 to 97 ms and a fork 6.7 ms; a list of millions
// would hold the GPU for minutes.
constexpr int64_t kMaxReserve = 1 << 16, kMaxList = 1 << 20;

// whether a * b, both positive, is less than `limit`
bool product_below(int64_t a, int64_t b, int64_t limit) { return a <= (limit - 1) / b; }

// The checks that attention and append share; fills pb.
int check_batch(const nq_paged_cache_t *c, const nq_paged_batch_t *b, int n_heads, const char *fn,
                PagedBatch *pb) {
    const std::string what(fn);
    if (!c || !b) return fail(NQ_INVALID_INPUT, what + ": NULL cache or batch");
    if (c->dtype != NQ_DTYPE_BF16 && c->dtype != NQ_DTYPE_F16)
        return fail(NQ_INVALID_INPUT, what + ": the cache is bf16 or fp16");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(NQ_INVALID_INPUT, what + ": head_dim must be 64, 128 or 256");
    if (c->n_kv_heads <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads)
        return fail(NQ_INVALID_INPUT, what + ": n_heads must be a positive multiple of n_kv_heads");
    if (c->page_size <= 0 || c->page_size % 16)
        return fail(NQ_INVALID_INPUT, what + ": page_size must be a positive multiple of 16");
    if (c->n_pages < 0 || c->n_pages >= kMaxInt || b->n_seqs < 0 || b->n_seqs >= kMaxInt ||
        b->n_tokens < 0 || b->n_tokens >= kMaxInt || b->n_rows < 0 || b->n_rows >= kMaxInt ||
        b->table_width < 0 || !product_below(b->table_width, c->page_size, kMaxInt) ||
        !product_below((int64_t)c->n_kv_heads * c->head_dim, c->page_size, (int64_t)1 << 62))
        return fail(NQ_INVALID_INPUT, what + ": a size is negative or too large");
    const int64_t page = (int64_t)c->n_kv_heads * c->page_size * c->head_dim;
    if (c->page_stride < page || c->page_stride % 8)
        return fail(NQ_INVALID_INPUT,
                    what + ": page_stride must be a multiple of 8 elements and hold a page");
    if (b->n_seqs == 0 || b->n_tokens == 0) return NQ_SUCCESS;
    if (!b->q_starts && b->n_tokens < b->n_seqs)
        return fail(NQ_INVALID_INPUT, what + ": without q_starts every entry is one token");
    if (b->n_rows == 0 || b->table_width == 0 || b->table_ld < b->table_width || c->n_pages == 0)
        return fail(NQ_INVALID_INPUT, what + ": empty table or cache");
    if (!b->seqs && b->n_seqs > b->n_rows)
        return fail(NQ_INVALID_INPUT, what + ": more entries than table rows");
    if (!c->k || !c->v || !b->table || !b->kv_lens)
        return fail(NQ_INVALID_INPUT, what + ": NULL cache, table or lengths");
    if (!aligned16(c->k) || !aligned16(c->v))
        return fail(NQ_INVALID_INPUT, what + ": the cache must be 16-byte aligned");
    pb->table = b->table;
    pb->lens = b->kv_lens;
    pb->seqs = b->seqs;
    pb->q_starts = b->q_starts;
    pb->table_ld = b->table_ld;
    pb->table_width = (int)b->table_width;
    pb->n_rows = (int)b->n_rows;
    pb->n_seqs = (int)b->n_seqs;
    pb->n_tokens = (int)b->n_tokens;
    pb->page_size = c->page_size;
    pb->n_pages = (int)c->n_pages;
    return NQ_SUCCESS;
}

int check_rows(const void *p, int64_t ld, int64_t heads, int hd, const char *fn, const char *name) {
    if (!p || !aligned16(p) || ld < heads * hd || ld % 8)
        return fail(NQ_INVALID_INPUT,
                    std::string(fn) + ": " + name +
                        " must be 16-byte aligned rows, a multiple of 8 elements apart");
    return NQ_SUCCESS;
}

int need_gpu(const char *fn) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        cudaGetLastError();
        return fail(NQ_BACKEND_NOT_AVAILABLE, std::string(fn) + ": no CUDA device");
    }
    return NQ_SUCCESS;
}

int check_table(const nq_page_table_t *t, int64_t n, int64_t most, const char *fn, PageTable *a) {
    const std::string what(fn);
    if (!t) return fail(NQ_INVALID_INPUT, what + ": NULL page table");
    if (n > most)
        return fail(NQ_INVALID_INPUT,
                    what + ": a list has at most " + std::to_string(most) + " entries");
    if (t->n_pages <= 0 || t->n_pages >= kMaxInt || t->n_rows <= 0 || t->n_rows >= kMaxInt ||
        t->table_width <= 0 || t->table_ld < t->table_width || t->page_size <= 0 ||
        !product_below(t->table_width, t->page_size, kMaxInt) || n < 0)
        return fail(NQ_INVALID_INPUT, what + ": a size is not positive or too large");
    if (!t->refs || !t->table || !t->lens)
        return fail(NQ_INVALID_INPUT, what + ": NULL refs, table or lens");
    a->refs = t->refs;
    a->table = t->table;
    a->lens = t->lens;
    a->table_ld = t->table_ld;
    a->table_width = (int)t->table_width;
    a->n_rows = (int)t->n_rows;
    a->n_pages = (int)t->n_pages;
    a->page_size = t->page_size;
    return NQ_SUCCESS;
}

int check_pool(const nq_page_pool_t *p, const char *fn, PagePool *a) {
    const std::string what(fn);
    if (!p || !p->data) return fail(NQ_INVALID_INPUT, what + ": NULL pool");
    if (p->outer <= 0 || p->n_pages <= 0 || p->n_pages >= kMaxInt || p->page_bytes <= 0 ||
        p->page_bytes % 16 || !aligned16(p->data))
        return fail(NQ_INVALID_INPUT,
                    what + ": the pool must be 16-byte aligned, its pages multiples of 16 bytes");
    a->data = static_cast<uint8_t *>(p->data);
    a->outer = p->outer;
    a->page_bytes = p->page_bytes;
    a->n_pages = (int)p->n_pages;
    return NQ_SUCCESS;
}

// workspace: move count (2 int32, padded), moves, then the plan's own arrays
Moves place_moves(void *ws) {
    Moves m;
    m.count = static_cast<int32_t *>(ws);
    m.pair = reinterpret_cast<int2 *>(static_cast<uint8_t *>(ws) + 256);
    return m;
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" {

size_t nq_paged_attention_workspace_size(int n_heads, int n_kv_heads, int head_dim, int64_t max_q,
                                         int64_t max_keys) {
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads ||
        n_heads / n_kv_heads > 128 || max_q < 0 || max_keys < 0 ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return 0;
    const size_t most = paged_attention_workspace(n_heads, n_kv_heads, head_dim, max_q, max_keys);
    // (a call with fewer new tokens may take the kernel that needs more)
    return max_q == 0 ? most
                      : std::max(most, paged_attention_workspace(n_heads, n_kv_heads, head_dim, 1,
                                                                 max_keys));
}

int nq_paged_attention(const uint16_t *q, int64_t q_ld, int n_heads, const nq_paged_cache_t *cache,
                       const nq_paged_batch_t *batch, int64_t max_q, float scale, int64_t window,
                       void *workspace, size_t workspace_bytes, uint16_t *out, int64_t out_ld,
                       void *stream) {
    const char *fn = "nq_paged_attention";
    const std::string what(fn);
    PagedAttnCall c{};
    if (int rc = check_batch(cache, batch, n_heads, fn, &c.pb)) return rc;
    if (n_heads / cache->n_kv_heads > 128)
        return fail(NQ_INVALID_INPUT, what + ": at most 128 query heads per key head");
    if (!(scale > 0.f) || !std::isfinite(scale))
        return fail(NQ_INVALID_INPUT, what + ": scale must be positive and finite");
    if (window < 0) return fail(NQ_INVALID_INPUT, what + ": window must not be negative");
    if (max_q < 0) return fail(NQ_INVALID_INPUT, what + ": max_q must not be negative");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return NQ_SUCCESS;
    if (int rc = check_rows(q, q_ld, n_heads, cache->head_dim, fn, "q")) return rc;
    if (int rc = check_rows(out, out_ld, n_heads, cache->head_dim, fn, "out")) return rc;
    if (int rc = need_gpu(fn)) return rc;
    c.max_q = !batch->q_starts ? 1 : (max_q == 0 ? batch->n_tokens : max_q);
    const size_t need =
        paged_attention_workspace(n_heads, cache->n_kv_heads, cache->head_dim, c.max_q,
                                  (int64_t)c.pb.table_width * c.pb.page_size);
    if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
                     workspace_bytes < need))
        return fail(NQ_INVALID_INPUT,
                    what + ": workspace must be 256-byte aligned and hold "
                           "nq_paged_attention_workspace_size() bytes");
    c.pb.err = device_error_word();
    c.q = q;
    c.k = static_cast<const uint16_t *>(cache->k);
    c.v = static_cast<const uint16_t *>(cache->v);
    c.out = out;
    c.q_ld = q_ld;
    c.out_ld = out_ld;
    c.page_stride = cache->page_stride;
    c.n_heads = n_heads;
    c.n_kv = cache->n_kv_heads;
    c.head_dim = cache->head_dim;
    // (a window as long as the table hides nothing)
    c.window = window < (int64_t)c.pb.table_width * c.pb.page_size ? (int)window : 0;
    c.f16 = cache->dtype == NQ_DTYPE_F16;
    c.scale = scale;
    c.ws = workspace;
    return from_cuda(launch_paged_attention(c, static_cast<cudaStream_t>(stream)), fn);
}

int nq_paged_append(const uint16_t *q, int64_t q_ld, const uint16_t *k, int64_t k_ld,
                    const uint16_t *v, int64_t v_ld, int n_heads, const nq_paged_cache_t *cache,
                    const nq_paged_batch_t *batch, const float *freqs, int n_freqs, uint16_t *q_out,
                    int64_t q_out_ld, void *stream) {
    const char *fn = "nq_paged_append";
    const std::string what(fn);
    AppendArgs a{};
    if (int rc = check_batch(cache, batch, n_heads, fn, &a.pb)) return rc;
    if (n_freqs < 0 || n_freqs % 8 || 2 * n_freqs > cache->head_dim || (n_freqs > 0 && !freqs))
        return fail(NQ_INVALID_INPUT,
                    what + ": freqs must be a multiple of 8 frequencies, at most head_dim / 2");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return NQ_SUCCESS;
    const int hd = cache->head_dim;
    if (int rc = check_rows(q, q_ld, n_heads, hd, fn, "q")) return rc;
    if (int rc = check_rows(k, k_ld, cache->n_kv_heads, hd, fn, "k")) return rc;
    if (int rc = check_rows(v, v_ld, cache->n_kv_heads, hd, fn, "v")) return rc;
    if (int rc = check_rows(q_out, q_out_ld, n_heads, hd, fn, "q_out")) return rc;
    if (int rc = need_gpu(fn)) return rc;
    a.pb.err = device_error_word();
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.kc = static_cast<uint16_t *>(cache->k);
    a.vc = static_cast<uint16_t *>(cache->v);
    a.freqs = freqs;
    a.q_ld = q_ld;
    a.k_ld = k_ld;
    a.v_ld = v_ld;
    a.q_out_ld = q_out_ld;
    a.page_stride = cache->page_stride;
    a.n_heads = n_heads;
    a.n_kv = cache->n_kv_heads;
    a.hd = hd;
    a.half = n_freqs;
    auto kern = cache->dtype == NQ_DTYPE_F16 ? paged_append_kernel<true> : paged_append_kernel<false>;
    return from_cuda(launch_pdl(kern, dim3((unsigned)batch->n_tokens), kAppendThreads, 0,
                                static_cast<cudaStream_t>(stream), a),
                     fn);
}

int nq_pages_free(const nq_page_table_t *table, const int32_t *seqs, int64_t n, void *stream) {
    const char *fn = "nq_pages_free";
    PageTable a{};
    if (int rc = check_table(table, n, kMaxList, fn, &a)) return rc;
    if (n == 0) return NQ_SUCCESS;
    if (!seqs) return fail(NQ_INVALID_INPUT, std::string(fn) + ": NULL list");
    if (int rc = need_gpu(fn)) return rc;
    a.err = device_error_word();
    return from_cuda(launch_pdl(pages_free_kernel, dim3((unsigned)n), 256, 0,
                                static_cast<cudaStream_t>(stream), a, seqs),
                     fn);
}

int nq_pages_fork(const nq_page_table_t *table, const int32_t *parents, const int32_t *children,
                  int64_t n, void *stream) {
    const char *fn = "nq_pages_fork";
    PageTable a{};
    if (int rc = check_table(table, n, kMaxList, fn, &a)) return rc;
    if (n == 0) return NQ_SUCCESS;
    if (!parents || !children) return fail(NQ_INVALID_INPUT, std::string(fn) + ": NULL list");
    if (int rc = need_gpu(fn)) return rc;
    a.err = device_error_word();
    return from_cuda(launch_pdl(pages_fork_kernel, dim3((unsigned)n), 256, 0,
                                static_cast<cudaStream_t>(stream), a, parents, children, (int)n),
                     fn);
}

size_t nq_pages_workspace_size(int64_t n_pages, int64_t n) {
    if (n_pages < 0 || n < 0) return 0;
    const size_t reserve = align256((size_t)n * sizeof(int2)) + (size_t)n * 3 * sizeof(int32_t);
    const size_t compact =
        align256((size_t)n_pages * sizeof(int2)) + (size_t)n_pages * sizeof(int32_t);
    return 256 + std::max(reserve, compact);
}

static int check_plan(const nq_page_table_t *table, const nq_page_pool_t *pool, int64_t n,
                      void *workspace, size_t bytes, size_t need, const char *fn, PageTable *a,
                      PagePool *p) {
    if (int rc = check_table(table, n, kMaxReserve, fn, a)) return rc;
    if (int rc = check_pool(pool, fn, p)) return rc;
    if (p->n_pages != a->n_pages)
        return fail(NQ_INVALID_INPUT, std::string(fn) + ": refs and the pool differ in pages");
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || bytes < need)
        return fail(NQ_INVALID_INPUT, std::string(fn) +
                                          ": workspace must be 256-byte aligned and hold "
                                          "nq_pages_workspace_size() bytes");
    if (int rc = need_gpu(fn)) return rc;
    a->err = device_error_word();
    return NQ_SUCCESS;
}

int nq_pages_reserve(const nq_page_table_t *table, const nq_page_pool_t *pool, const int32_t *seqs,
                     const int32_t *new_lens, int64_t n, void *workspace, size_t workspace_bytes,
                     void *stream) {
    const char *fn = "nq_pages_reserve";
    PageTable a{};
    PagePool p{};
    // (the plan counts the pages that the list can ask for in 32 bits)
    if (table && n > 0 && n <= kMaxReserve && table->table_width < kMaxInt &&
        n * table->table_width >= kMaxInt)
        return fail(NQ_INVALID_INPUT, std::string(fn) + ": a size is not positive or too large");
    if (int rc = check_plan(table, pool, n, workspace, workspace_bytes,
                            nq_pages_workspace_size(0, n), fn, &a, &p))
        return rc;
    if (n == 0) return NQ_SUCCESS;
    if (!seqs || !new_lens) return fail(NQ_INVALID_INPUT, std::string(fn) + ": NULL list");
    const Moves mv = place_moves(workspace);
    int32_t *ws = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(workspace) + 256 +
                                              align256((size_t)n * sizeof(int2)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_pdl(pages_reserve_kernel, dim3(1), kPlanThreads, 0, st, a, seqs,
                               new_lens, (int)n, ws, mv);
    if (e == cudaSuccess)
        e = launch_pdl(pages_move_kernel, dim3((unsigned)(sm_count() * 8)), kCopyThreads, 0, st, p,
                       mv, a, (const int32_t *)nullptr);
    return from_cuda(e, fn);
}

int nq_pages_compact(const nq_page_table_t *table, const nq_page_pool_t *pool, void *workspace,
                     size_t workspace_bytes, void *stream) {
    const char *fn = "nq_pages_compact";
    PageTable a{};
    PagePool p{};
    if (int rc = check_plan(table, pool, 0, workspace, workspace_bytes,
                            table ? nq_pages_workspace_size(table->n_pages, 0) : 0, fn, &a, &p))
        return rc;
    const Moves mv = place_moves(workspace);
    int32_t *to = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(workspace) + 256 +
                                              align256((size_t)a.n_pages * sizeof(int2)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_pdl(pages_compact_kernel, dim3(1), kPlanThreads, 0, st, a, to, mv);
    if (e == cudaSuccess)
        e = launch_pdl(pages_move_kernel, dim3((unsigned)(sm_count() * 8)), kCopyThreads, 0, st, p,
                       mv, a, (const int32_t *)to);
    return from_cuda(e, fn);
}

int nq_pages_copy(const nq_page_pool_t *pool, const int32_t *src, const int32_t *dst, int64_t n,
                  void *stream) {
    const char *fn = "nq_pages_copy";
    PagePool p{};
    if (int rc = check_pool(pool, fn, &p)) return rc;
    if (n < 0 || n > kMaxList)
        return fail(NQ_INVALID_INPUT, std::string(fn) + ": a list has at most " +
                                          std::to_string(kMaxList) + " entries");
    if (n == 0) return NQ_SUCCESS;
    if (!src || !dst) return fail(NQ_INVALID_INPUT, std::string(fn) + ": NULL list");
    if (int rc = need_gpu(fn)) return rc;
    const int64_t pieces = p.outer * ((p.page_bytes + kCopyBytes - 1) / kCopyBytes);
    const unsigned gx = (unsigned)std::min<int64_t>(n, 65535);
    const unsigned gy = (unsigned)std::min<int64_t>(
        pieces, std::max<int64_t>(1, ((int64_t)sm_count() * 8 + gx - 1) / gx));
    return from_cuda(launch_pdl(pages_copy_kernel, dim3(gx, gy), kCopyThreads, 0,
                                static_cast<cudaStream_t>(stream), p, src, dst, (int)n,
                                device_error_word()),
                     fn);
}

}  // extern "C"
