// attn_paged.cu -- attention of new tokens over the paged cache, for few query
// rows per key head (a decode step), and the merge of tiles that several CTAs
// share.  attn_paged_tc.cu holds the kernel for many rows.
//
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,   p_j = exp(scale q[t, h] . k[j, h / G])
// over the keys j <= pos(t) = len - n + t (and j > pos(t) - window), G query
// heads per key head.
//
// A tile is 16 rows: the G query heads of a key head times 16 / G tokens, the
// M of an m16n8k16 MMA, so that each key and value is read from memory once
// for all of them.  The call's key blocks (64 keys) are dealt out evenly over
// the CTAs (paged.cuh); per CTA one warp brings blocks into a ring of
// shared-memory stages by TMA (16- to 64-row boxes, as the page size allows),
// and four warps take 16 keys of each block: S = Q K^T, a running maximum and
// sum per row, O += P V, all in registers, without a barrier between the
// warps until the tile's end.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "nq_common.cuh"
#include "nq_internal.h"
#include "paged.cuh"

namespace nq {
namespace {

constexpr int kRows = 16;          // query rows per tile
constexpr int kBlock = 64;         // keys per block
constexpr int kWarps = 4;          // consumer warps, 16 keys of a block each
constexpr int kThreads = 32 * (kWarps + 1);

template <int HD>
struct Cfg {
    static constexpr int kTileBytes = kBlock * HD * 2;   // keys (or values) of a block
    static constexpr int kStageBytes = 2 * kTileBytes;
    // two CTAs per SM at 64 and 128 dims, one at 256: 96 to 128 KB of loads in
    // flight per SM, where 6.5 TB/s and about 1 us of latency ask for 44 KB
    static constexpr int kStages = HD == 64 ? 5 : (HD == 128 ? 3 : 2);
    static constexpr int kRedBytes = 2 * kRows * HD * 4;  // two warps' O at a tile's end
    static constexpr int kSmem = kStages * kStageBytes + kRedBytes;
    static constexpr int kCtas = HD == 256 ? 1 : 2;  // per SM
};

template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    if constexpr (F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Loads key block `blk` (keys and values) of a piece into one stage: boxes of
// `box` keys x 64 dims, one lane each.  Boxes without a visible key of the
// piece read as zeros through a coordinate outside of the tensor (their pages
// need not exist).
template <int HD>
__device__ __forceinline__ void load_block(const PagedBatch &pb, const CUtensorMap *mk,
                                           const CUtensorMap *mv, const Piece &p, int blk, int box,
                                           int key_lo, int key_hi, uint8_t *stage, uint64_t *bar) {
    constexpr int kCols = HD / 64;
    const int lane = threadIdx.x & 31;
    const int per = kBlock / box * kCols;  // boxes of the keys; as many of the values
    const bool is_v = lane >= per;
    const int i = is_v ? lane - per : lane;
    const int r = i / kCols, col = i % kCols;
    const int key = blk * kBlock + r * box;
    int page = pb.n_pages, slot = 0;
    if (lane < 2 * per && key < key_hi && key + box > key_lo) {
        page = page_of(pb, p.s.row, key);
        slot = key % pb.page_size;
    }
    if (lane == 0) mbar_expect_tx(bar, Cfg<HD>::kStageBytes);
    __syncwarp();
    if (lane < 2 * per)
        tma_load_4d(stage + (is_v ? Cfg<HD>::kTileBytes : 0) + col * (kBlock * 128) + r * box * 128,
                    is_v ? mv : mk, bar, col * 64, slot, p.h, page);
}

template <int HD, bool F16>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kCtas) paged_rows_kernel(
    const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
    const PagedAttnArgs a) {
    using C = Cfg<HD>;
    extern __shared__ __align__(1024) uint8_t smem[];  // (the swizzle's period)
    float *red = reinterpret_cast<float *>(smem + C::kStages * C::kStageBytes);
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages];
    __shared__ float wm[kWarps][kRows], wl[kWarps][kRows];
    __shared__ int abort_flag, stop;
    volatile int *abort = &abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.n_heads / a.n_kv, TT = kRows / G;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
        abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    __syncthreads();
    pdl_wait();  // lengths, tables, q and the cache come from earlier kernels

    const Share sh = find_share<kBlock>(a.pb, a.n_kv, TT, a.window, blockIdx.x, gridDim.x, a.least,
                                        a.whole);
    Cursor c = sh.c;
    int64_t unit = sh.first;
    Piece p;
    int it = 0;  // blocks so far: stage it % kStages, parity it / kStages

    if (warp == kWarps) {
        while (next_piece<kBlock>(a.pb, a.n_kv, TT, a.window, a.whole, c, p)) {
            const int p0 = p.s.len - p.s.n + p.t0, key_hi = p.s.len - p.s.n + p.t1;
            const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
            for (int k = p.k0; k < p.k1; ++k, ++it) {
                const int st = it % C::kStages;
                if (!mbar_wait_or_abort(&empty[st], (uint32_t)(it / C::kStages + 1) & 1u, abort,
                                        a.pb.err)) {
                    // given up: the copies in flight end before this CTA does
                    for (int j = max(0, it - C::kStages); j < it; ++j) {
                        const unsigned long long t0 = global_timer_ns();
                        while (!mbar_try_wait(&full[j % C::kStages],
                                              (uint32_t)(j / C::kStages) & 1u) &&
                               global_timer_ns() - t0 < kWaitLimitNs) {
                        }
                    }
                    return;
                }
                load_block<HD>(a.pb, &mk, &mv, p, p.lo + k, a.box, key_lo, key_hi,
                               smem + st * C::kStageBytes, &full[st]);
            }
        }
        return;  // (the consumers wait for every load)
    }

    const float cs = a.scale * 1.4426950408889634f;  // exp(scale x) = 2^(cs x)
    const int r0 = lane >> 2, cq = (lane & 3) * 2;   // rows r0, r0 + 8; columns cq, cq + 1 (+ 8)
    bool note_left = false;
    while (next_piece<kBlock>(a.pb, a.n_kv, TT, a.window, a.whole, c, p)) {
        const int valid = (p.t1 - p.t0) * G;
        const int base = p.s.len - p.s.n;            // position of the first new token
        const int p0 = base + p.t0, key_hi = base + p.t1;
        const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
        int pos[2];
        uint32_t qf[HD / 16][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            const bool in = r < valid;
            const int t = p.t0 + (in ? r / G : 0);
            pos[i] = in ? base + t : -1;
            const uint16_t *qp =
                a.q + (int64_t)(p.s.q0 + t) * a.q_ld + (int64_t)(p.h * G + (in ? r % G : 0)) * HD;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                qf[k][i] = in ? *reinterpret_cast<const uint32_t *>(qp + k * 16 + cq) : 0u;
                qf[k][i + 2] = in ? *reinterpret_cast<const uint32_t *>(qp + k * 16 + cq + 8) : 0u;
            }
        }
        float o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][j] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        for (int k = p.k0; k < p.k1; ++k, ++it) {
            const int st = it % C::kStages;
            const int key0 = (p.lo + k) * kBlock + warp * 16;  // this warp's keys
            // (given up: the warp still takes part in the barriers below)
            if (!mbar_wait_or_abort(&full[st], (uint32_t)(it / C::kStages) & 1u, abort, a.pb.err))
                break;
            if (key0 < key_hi && key0 + 16 > key_lo) {
                uint8_t *ks = smem + st * C::kStageBytes + warp * 16 * 128;
                uint8_t *vs = ks + C::kTileBytes;
                float s[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
                {
                    // matrices: keys 0-7 / dims 0-7, keys 0-7 / dims 8-15, then keys 8-15
                    const int row = (lane & 7) + ((lane >> 4) << 3);
                    const uint32_t rowa = smem_u32(ks) + row * 128;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const int ch = (kk & 3) * 2 + ((lane >> 3) & 1);
                        uint32_t b[4];
                        ldsm4(b, rowa + (kk >> 2) * (kBlock * 128) + ((ch ^ (row & 7)) << 4));
                        mma16816<F16>(s[0], qf[kk], b[0], b[1]);
                        mma16816<F16>(s[1], qf[kk], b[2], b[3]);
                    }
                }
                if (key0 + 15 > p0 || (a.window > 0 && key0 <= key_hi - 1 - a.window)) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = key0 + n * 8 + cq + (j & 1), ps = pos[j >> 1];
                            if (key > ps || (a.window > 0 && key <= ps - a.window))
                                s[n][j] = -INFINITY;
                        }
                }
                if (key0 < key_lo || key0 + 16 > key_hi) {
                    // values of keys that no row sees may hold anything: a NaN times
                    // a weight of 0 would reach the sum
#pragma unroll
                    for (int i = lane; i < 16 * (HD / 8); i += 32) {
                        const int row = i & 15, cc = i >> 4;
                        const int key = key0 + row;
                        if (key < key_lo || key >= key_hi)
                            *reinterpret_cast<uint4 *>(vs + (cc >> 3) * (kBlock * 128) + row * 128 +
                                                       (cc & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                // running maximum and sum of rows r0 and r0 + 8, in fp32
                float mn[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float x = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]),
                                    fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    mn[i] = fmaxf(m[i], x);
                }
                if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float f = m[i] == -INFINITY ? 0.f : ex2((m[i] - mn[i]) * cs);
                        l[i] *= f;
#pragma unroll
                        for (int n = 0; n < HD / 8; ++n) {
                            o[n][2 * i] *= f;
                            o[n][2 * i + 1] *= f;
                        }
                        m[i] = mn[i];
                    }
                }
                uint32_t pf[4];
                {
                    const float z[2] = {m[0] == -INFINITY ? 0.f : m[0] * cs,
                                        m[1] == -INFINITY ? 0.f : m[1] * cs};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float e0 = ex2(fmaf(s[n][2 * i], cs, -z[i]));
                            const float e1 = ex2(fmaf(s[n][2 * i + 1], cs, -z[i]));
                            l[i] += e0 + e1;
                            // the weights are rounded to the cache's type, as the
                            // tensor cores take both factors in one type
                            pf[n * 2 + i] = pack_t2<F16>(e0, e1);
                        }
                }
                {
                    // matrices: keys 0-7 and 8-15 of dims 0-7, then of dims 8-15
                    const int row = lane & 15;
                    const uint32_t rowa = smem_u32(vs) + row * 128;
#pragma unroll
                    for (int n = 0; n < HD / 16; ++n) {
                        const int ch = (n & 3) * 2 + (lane >> 4);
                        uint32_t b[4];
                        ldsm4_t(b, rowa + (n >> 2) * (kBlock * 128) + ((ch ^ (row & 7)) << 4));
                        mma16816<F16>(o[2 * n], pf, b[0], b[1]);
                        mma16816<F16>(o[2 * n + 1], pf, b[2], b[3]);
                    }
                }
                if (key0 < key_lo || key0 + 16 > key_hi) fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }

        // the four warps' sums, one after another in a fixed order
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) {
                wm[warp][r0 + 8 * i] = m[i];
                wl[warp][r0 + 8 * i] = l[i];
            }
        }
        bar_sync(1, kWarps * 32);
        float M[2], L[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            M[i] = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
            L[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                L[i] += wm[w][r] == -INFINITY ? 0.f : wl[w][r] * ex2((wm[w][r] - M[i]) * cs);
            const float f = m[i] == -INFINITY ? 0.f : ex2((m[i] - M[i]) * cs);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                o[n][2 * i] *= f;
                o[n][2 * i + 1] *= f;
            }
        }
        float *mine = red + (warp & 1) * (kRows * HD);
        if (warp >= 2) {
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) mine[(n * 4 + j) * 32 + lane] = o[n][j];
        }
        bar_sync(1, kWarps * 32);
        if (warp < 2) {
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[n][j] += mine[(n * 4 + j) * 32 + lane];
                    if (warp == 1) mine[(n * 4 + j) * 32 + lane] = o[n][j];
                }
        }
        bar_sync(1, kWarps * 32);
        if (warp == 0) {
            const float *other = red + kRows * HD;
            const bool whole = p.k0 == 0 && p.k1 == p.nb;
            const int slot = 2 * blockIdx.x + (p.k0 == 0 ? 1 : 0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = r0 + 8 * i;
                if (r >= valid) continue;
                const float f = whole ? (L[i] == 0.f ? 0.f : 1.f / L[i]) : 1.f;
                uint16_t *op = a.out + (int64_t)(p.s.q0 + p.t0 + r / G) * a.out_ld +
                               (int64_t)(p.h * G + r % G) * HD;
                float *pp = a.part_o + ((int64_t)slot * kRows + r) * HD;
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) {
                    const float x = (o[n][2 * i] + other[(n * 4 + 2 * i) * 32 + lane]) * f;
                    const float y = (o[n][2 * i + 1] + other[(n * 4 + 2 * i + 1) * 32 + lane]) * f;
                    if (whole)
                        *reinterpret_cast<uint32_t *>(op + n * 8 + cq) = pack_t2<F16>(x, y);
                    else
                        *reinterpret_cast<float2 *>(pp + n * 8 + cq) = make_float2(x, y);
                }
                if (!whole && (lane & 3) == 0) {
                    float *ml = a.part_ml + ((int64_t)slot * kRows + r) * 2;
                    ml[0] = M[i] * cs;
                    ml[1] = L[i];
                }
            }
            if (!whole && p.k0 == 0) {
                note_left = true;
                if (lane == 0)
                    a.notes[blockIdx.x] = SplitNote{
                        p.s.q0 + p.t0, p.h * G, p.t1 - p.t0,
                        share_owner(sh.total, sh.n, unit + p.nb - 1) - (int)blockIdx.x + 1};
            }
            if (lane == 0) stop = *abort;
        }
        bar_sync(1, kWarps * 32);
        if (stop) break;  // one decision for all four warps
        unit += p.k1 - p.k0;
    }
    if (warp == 0 && lane == 0 && !note_left && !a.whole) a.notes[blockIdx.x] = SplitNote{0, 0, 0, 0};
}

// Joins the parts of the tiles that several CTAs shared, in the CTAs' order:
// one warp per query row.
template <int HD, bool F16>
__global__ void __launch_bounds__(128) paged_merge_kernel(const PagedAttnArgs a, int rows) {
    pdl_launch_dependents();
    pdl_wait();
    const SplitNote note = a.notes[blockIdx.x];
    if (note.parts == 0) return;
    const int G = a.n_heads / a.n_kv;
    const int r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= note.tokens * G) return;
    constexpr int kPer = HD / 32;
    auto slot = [&](int i) -> int64_t {
        return (int64_t)(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * rows + r;
    };
    float M = -INFINITY;
    for (int i = lane; i < note.parts; i += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + slot(i) * 2);
        if (ml.y != 0.f) M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float L = 0.f, acc[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
#pragma unroll 4
    for (int i = 0; i < note.parts; ++i) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + slot(i) * 2);
        const float *po = a.part_o + slot(i) * HD + lane * kPer;
        float v[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j += 2) {
            const float2 w = *reinterpret_cast<const float2 *>(po + j);
            v[j] = w.x;
            v[j + 1] = w.y;
        }
        const float f = ml.y != 0.f ? ex2(ml.x - M) : 0.f;
        L += ml.y * f;
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = fmaf(v[j], f, acc[j]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t *op = a.out + (int64_t)(note.q_row + r / G) * a.out_ld +
                   (int64_t)(note.heads0 + r % G) * HD + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; j += 2)
        *reinterpret_cast<uint32_t *>(op + j) = pack_t2<F16>(acc[j] * inv, acc[j + 1] * inv);
}

// CTAs of paged_rows_kernel: as many as fit at once
int rows_grid(int hd) { return sm_count() * (hd == 256 ? Cfg<256>::kCtas : Cfg<128>::kCtas); }

// Which kernel serves a call: paged_rows_kernel while a sequence's new tokens
// make one tile of 16 rows, so that each key is read once; the tensor-core
// kernel (128- or 256-row tiles) from there on.
// A table that holds at most kWholeKeys keys per sequence leaves the tiles whole.
struct Shape {
    bool tiles, whole;
    int grid, rows, block;  // CTAs, rows of a part, keys of a block
};

constexpr int64_t kWholeKeys = 512;

Shape shape_of(int n_heads, int n_kv, int hd, int64_t max_q, int64_t max_keys) {
    const int G = n_heads / n_kv;
    const bool whole = max_keys <= kWholeKeys;
    if (max_q * G > kRows) return Shape{true, whole, sm_count(), paged_tiles_rows(hd), 128};
    return Shape{false, whole, rows_grid(hd), kRows, kBlock};
}

template <int HD, bool F16>
cudaError_t run_rows(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                     cudaStream_t st) {
    auto kern = paged_rows_kernel<HD, F16>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, Cfg<HD>::kSmem, allowed);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3((unsigned)rows_grid(HD)), kThreads, Cfg<HD>::kSmem, st, mk, mv, a);
}

template <int HD, bool F16>
cudaError_t run_attention(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                          const Shape &s, cudaStream_t st) {
    const cudaError_t e = s.tiles ? launch_paged_tiles(a, mk, mv, HD, F16, st)
                                  : run_rows<HD, F16>(a, mk, mv, st);
    if (e != cudaSuccess || s.whole) return e;
    return launch_pdl(paged_merge_kernel<HD, F16>, dim3((unsigned)s.grid, (unsigned)s.rows / 4),
                      128, 0, st, a, s.rows);
}

// A workspace holds, for each CTA, the note and two parts of `rows` rows.
size_t part_bytes(int grid, int rows, int hd) {
    return align256((size_t)grid * sizeof(SplitNote)) +
           align256((size_t)2 * grid * rows * 2 * sizeof(float)) +
           (size_t)2 * grid * rows * hd * sizeof(float);
}

void place_workspace(PagedAttnArgs &a, int grid, int rows, void *ws) {
    uint8_t *p = static_cast<uint8_t *>(ws);
    a.notes = reinterpret_cast<SplitNote *>(p);
    p += align256((size_t)grid * sizeof(SplitNote));
    a.part_ml = reinterpret_cast<float *>(p);
    p += align256((size_t)2 * grid * rows * 2 * sizeof(float));
    a.part_o = reinterpret_cast<float *>(p);
}

}  // namespace

size_t paged_attention_workspace(int n_heads, int n_kv, int head_dim, int64_t max_q,
                                 int64_t max_keys) {
    const Shape s = shape_of(n_heads, n_kv, head_dim, max_q, max_keys);
    return s.whole ? 0 : part_bytes(s.grid, s.rows, head_dim);
}

cudaError_t launch_paged_attention(const PagedAttnCall &c, cudaStream_t st) {
    const Shape s = shape_of(c.n_heads, c.n_kv, c.head_dim, c.max_q,
                             (int64_t)c.pb.table_width * c.pb.page_size);
    PagedAttnArgs a;
    a.pb = c.pb;
    a.q = c.q;
    a.q_ld = c.q_ld;
    a.out = c.out;
    a.out_ld = c.out_ld;
    a.n_heads = c.n_heads;
    a.n_kv = c.n_kv;
    a.window = c.window;
    a.scale = c.scale;
    a.least = 1;
    a.whole = s.whole;
    // the largest power of two that divides the page size: no box crosses a page
    a.box = std::min(s.block, c.pb.page_size & -c.pb.page_size);
    if (!s.whole) place_workspace(a, s.grid, s.rows, c.ws);
    CUtensorMap mk, mv;
    if (!make_map_pages(&mk, c.f16, c.k, c.head_dim, c.pb.page_size, c.n_kv, c.pb.n_pages,
                        c.page_stride, a.box) ||
        !make_map_pages(&mv, c.f16, c.v, c.head_dim, c.pb.page_size, c.n_kv, c.pb.n_pages,
                        c.page_stride, a.box))
        return cudaErrorInvalidValue;
    if (c.f16) {
        if (c.head_dim == 64) return run_attention<64, true>(a, mk, mv, s, st);
        if (c.head_dim == 128) return run_attention<128, true>(a, mk, mv, s, st);
        return run_attention<256, true>(a, mk, mv, s, st);
    }
    if (c.head_dim == 64) return run_attention<64, false>(a, mk, mv, s, st);
    if (c.head_dim == 128) return run_attention<128, false>(a, mk, mv, s, st);
    return run_attention<256, false>(a, mk, mv, s, st);
}

}  // namespace nq
