// attn_paged.cu -- attention of new tokens over the paged cache, for few query
// rows per key head (a decode step), and the merge of tiles that several CTAs
// share.  attn_paged_tc.cu holds the kernel for many rows.
//
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,   p_j = exp(scale q[t, h] . k[j, h / G])
// over the keys j <= pos(t) = len - n + t (and j > pos(t) - window), G query
// heads per key head.
//
// A tile is up to 8 or 16 rows: the G query heads of a key head times as many
// tokens as fit, so that each key and value is read from memory once for all of
// them.  The products are taken transposed, S^T = K Q^T and O^T += V^T P^T, with
// the keys (and dims) as the 16 rows of m16n8k16 and the query rows as its 8
// columns: a decode step with G <= 8 pays half of the MMAs and registers that
// 16 query rows would cost.  The call's key blocks (64 keys) are dealt out
// evenly over the CTAs (paged.cuh); per CTA one warp brings blocks into a ring
// of shared-memory stages by TMA (16- to 64-row boxes, as the page size
// allows), and four warps take 16 keys of each block, with a running maximum
// and sum of their own, all in registers, without a barrier between the warps
// until the tile's end.
//
// Bounded by HBM where there are many keys: 64 sequences of up to 8192 keys (554
// MB) 95 us, 5.8 TB/s or 0.89 of a copy's rate; two of 100003 and 61805 (331 MB)
// 60 us, 0.84; the rest is the start (about 4 us until a CTA's first keys are
// there: lengths, table and keys are one memory trip after another) and the merge
// (2 us).  One token over 200 keys, 7.3 us, is these trips alone where the table
// has room for 256 keys at most; in a wider one (any server's) its tiles are cut
// and joined, 10.4 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "nq_common.cuh"
#include "nq_internal.h"
#include "paged.cuh"

namespace nq {
namespace {

constexpr int kBlock = 64;         // keys per block
constexpr int kWarps = 4;          // consumer warps, 16 keys of a block each
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kRows = 16;          // query rows of a tile at most (8 NT)

template <int HD>
struct Cfg {
    static constexpr int kTileBytes = kBlock * HD * 2;   // keys (or values) of a block
    static constexpr int kStageBytes = 2 * kTileBytes;
    // 128 to 192 KB of loads in flight per SM, where 6.5 TB/s and about 1 us of
    // latency ask for 44 KB
    static constexpr int kCtas = HD == 64 ? 3 : (HD == 128 ? 2 : 1);  // per SM
    static constexpr int kStages = HD == 64 ? 4 : (HD == 128 ? 3 : 2);
    static constexpr int kRedBytes = kWarps * 8 * HD * 4;  // the warps' O of 8 rows
    static constexpr int kSmem = kStages * kStageBytes + kRedBytes;
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

// transposes an 8 x 8 matrix of 16-bit values held two per lane
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Loads key block `blk` (keys and values) of a piece into one stage: boxes of
// `box` keys x all dims (as columns of 64 dims, one after another), one lane
// each.  An SM starts a box about every 40 ns, which is why they are as large
// as the page size allows (64 keys: 0.6 us, 16 keys x 64 dims: 1.05 us a block
// where one CTA works alone).  Boxes without a visible key of the piece read as
// zeros through a coordinate outside of the tensor (their pages need not
// exist).
template <int HD>
__device__ __forceinline__ void load_block(const PagedBatch &pb, const CUtensorMap *mk,
                                           const CUtensorMap *mv, const Piece &p, int blk, int box,
                                           int key_lo, int key_hi, uint8_t *stage, uint64_t *bar) {
    const int lane = threadIdx.x & 31;
    const int per = kBlock / box;  // boxes of the keys; as many of the values
    const bool is_v = lane >= per;
    const int r = is_v ? lane - per : lane;
    const int key = blk * kBlock + r * box;
    int page = pb.n_pages, slot = 0;
    if (lane < 2 * per && key < key_hi && key + box > key_lo) {
        page = page_of(pb, p.s.row, key);
        slot = key % pb.page_size;
    }
    if (lane == 0) mbar_expect_tx(bar, Cfg<HD>::kStageBytes);
    __syncwarp();
    if (lane < 2 * per)
        tma_load_5d(stage + (is_v ? Cfg<HD>::kTileBytes : 0) + r * box * HD * 2, is_v ? mv : mk, bar,
                    0, slot, 0, p.h, page);
}

// Q^T as the MMAs' second operand: lane l holds query row l / 4 (+ 8), dims
// (l % 4) * 2 + {0, 1} (+ 8) of each 16.
template <int HD, int NT>
__device__ __forceinline__ void load_q(const PagedAttnArgs &a, const Piece &p, int G,
                                       uint32_t (&q)[HD / 16][NT][2]) {
    const int lane = threadIdx.x & 31;
    const int valid = (p.t1 - p.t0) * G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + (lane >> 2);
        const bool in = r < valid;
        const uint16_t *src = a.q + (int64_t)(p.s.q0 + p.t0 + (in ? r / G : 0)) * a.q_ld +
                              (int64_t)(p.h * G + (in ? r % G : 0)) * HD + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            q[k][nt][0] = in ? *reinterpret_cast<const uint32_t *>(src + k * 16) : 0u;
            q[k][nt][1] = in ? *reinterpret_cast<const uint32_t *>(src + k * 16 + 8) : 0u;
        }
    }
}

template <int HD, bool F16, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kCtas) paged_rows_kernel(
    const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
    const PagedAttnArgs a) {
    using C = Cfg<HD>;
    // the next tile's queries are loaded while this one's keys are worked on,
    // where registers allow
    constexpr bool kAhead = HD / 16 * NT <= 8;
    extern __shared__ __align__(1024) uint8_t smem[];  // (the swizzle's period)
    float *red = reinterpret_cast<float *>(smem + C::kStages * C::kStageBytes);
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages];
    __shared__ float wm[kWarps][8 * NT], wl[kWarps][8 * NT];
    __shared__ int abort_flag, stop;
    volatile int *abort = &abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.n_heads / a.n_kv, TT = 8 * NT / G;

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

    const Tiling tl{TT, TT, a.window, a.whole};
    Share sh = find_share<kBlock>(a.pb, a.n_kv, tl, blockIdx.x, gridDim.x);
    Piece p;
    int it = 0;  // blocks so far: stage it % kStages, parity it / kStages

    if (warp == kWarps) {
        while (next_piece<kBlock>(a.pb, a.n_kv, tl, sh, blockIdx.x, p)) {
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
        return;  // (the consumers wait for every load, or below)
    }

    const float cs = a.scale * 1.4426950408889634f;  // exp(scale x) = 2^(cs x)
    const int kr = lane >> 2, cq = (lane & 3) * 2;   // keys kr, kr + 8; rows cq, cq + 1 (+ 8 nt)
    // this warp's 16 keys in a stage, and the distance of the columns of 64 dims
    const int key_at = warp * 16 / a.box * a.box * (HD * 2) + warp * 16 % a.box * 128;
    const int col_ld = a.box * 128;
    bool note_left = false;
    uint32_t q[HD / 16][NT][2], qn[kAhead ? HD / 16 : 1][NT][2];
    Piece pn;
    bool more = next_piece<kBlock>(a.pb, a.n_kv, tl, sh, blockIdx.x, pn);
    if constexpr (kAhead) {
        if (more) load_q<HD, NT>(a, pn, G, qn);
    }
    while (more) {
        p = pn;
        if constexpr (kAhead) {
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) q[k][nt][e] = qn[k][nt][e];
        } else {
            load_q<HD, NT>(a, p, G, q);
        }
        more = next_piece<kBlock>(a.pb, a.n_kv, tl, sh, blockIdx.x, pn);
        if constexpr (kAhead) {
            if (more) load_q<HD, NT>(a, pn, G, qn);
        }
        const int valid = (p.t1 - p.t0) * G;
        const int base = p.s.len - p.s.n;            // position of the first new token
        const int p0 = base + p.t0, key_hi = base + p.t1;
        const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
        int pos[NT][2];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nt * 8 + cq + e;
                pos[nt][e] = r < valid ? p0 + r / G : -1;
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
            }
        float o[HD / 16][NT][4];
#pragma unroll
        for (int t = 0; t < HD / 16; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t][nt][j] = 0.f;

        for (int k = p.k0; k < p.k1; ++k, ++it) {
            const int st = it % C::kStages;
            const int key0 = (p.lo + k) * kBlock + warp * 16;  // this warp's keys
            // (given up: the warp still takes part in the barriers below)
            if (!warp_wait_or_abort(&full[st], (uint32_t)(it / C::kStages) & 1u, abort, a.pb.err))
                break;
            if (key0 < key_hi && key0 + 16 > key_lo) {
                uint8_t *ks = smem + st * C::kStageBytes + key_at;
                uint8_t *vs = ks + C::kTileBytes;
                // two chains of sums over the dims, so that an MMA waits for the last
                // but one
                float s[NT][4], s2[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[nt][j] = s2[nt][j] = 0.f;
                {
                    // matrices: keys 0-7 / dims 0-7, keys 8-15 / dims 0-7, then dims 8-15
                    const int row = lane & 15;
                    const uint32_t rowa = smem_u32(ks) + row * 128;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const int ch = (kk & 3) * 2 + (lane >> 4);
                        uint32_t f[4];
                        ldsm4(f, rowa + (kk >> 2) * col_ld + ((ch ^ (row & 7)) << 4));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16816<F16>((kk & 1) ? s2[nt] : s[nt], f, q[kk][nt][0], q[kk][nt][1]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[nt][j] += s2[nt][j];
                }
                if (key0 + 15 > p0 || (a.window > 0 && key0 <= key_hi - 1 - a.window)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = key0 + kr + (j >> 1) * 8, ps = pos[nt][j & 1];
                            if (key > ps || (a.window > 0 && key <= ps - a.window))
                                s[nt][j] = -INFINITY;
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
                            *reinterpret_cast<uint4 *>(vs + (cc >> 3) * col_ld + row * 128 +
                                                       (cc & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                // Running maximum and sum of each row (a column here), in fp32.  The
                // maximum follows only when a score has passed it by 2^8 (or the row has
                // none yet): until then weights up to 2^8 do no harm, and the warp is
                // spared the maximum over its lanes.
                bool grow = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        grow |= (fmaxf(s[nt][e], s[nt][e + 2]) - m[nt][e]) * cs > 8.f;
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1)
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            x = fmaxf(x, m[nt][e]);
                            const float f =
                                m[nt][e] == -INFINITY ? 0.f : ex2((m[nt][e] - x) * cs);
                            m[nt][e] = x;
                            l[nt][e] *= f;
#pragma unroll
                            for (int t = 0; t < HD / 16; ++t) {
                                o[t][nt][e] *= f;
                                o[t][nt][e + 2] *= f;
                            }
                        }
                }
                // The weights go to the tensor cores, which take both factors in one type, as
                // two terms of it, a weight's rounding and what that left out: 16 bits of
                // precision or more, where one term made a result's error 1.4 times that of
                // its own rounding.  (The tensor pipe, 10 % busy with one term, is 15 % busy
                // with two: 64 sequences 94.8 -> 95.2 us, one token over 200 keys 7.21 ->
                // 7.31.)
                uint32_t pf[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float z = m[nt][e] == -INFINITY ? 0.f : m[nt][e] * cs;
                        w[e] = ex2(fmaf(s[nt][e], cs, -z));
                        w[e + 2] = ex2(fmaf(s[nt][e + 2], cs, -z));
                        l[nt][e] += w[e] + w[e + 2];
                    }
                    const uint32_t h0 = pack_t2<F16>(w[0], w[1]), h1 = pack_t2<F16>(w[2], w[3]);
                    pf[nt][0] = transpose8(h0);
                    pf[nt][1] = transpose8(h1);
                    pl[nt][0] = transpose8(pack_t2<F16>(w[0] - t16_to_f32<F16>((uint16_t)h0),
                                                        w[1] - t16_to_f32<F16>((uint16_t)(h0 >> 16))));
                    pl[nt][1] = transpose8(pack_t2<F16>(w[2] - t16_to_f32<F16>((uint16_t)h1),
                                                        w[3] - t16_to_f32<F16>((uint16_t)(h1 >> 16))));
                }
                {
                    // matrices: dims 0-7 / keys 0-7, dims 8-15 / keys 0-7, then keys 8-15;
                    // four dims' products between the two that add to the same sums
                    const int row = (lane & 7) + ((lane >> 4) << 3);
                    const uint32_t rowa = smem_u32(vs) + row * 128;
#pragma unroll
                    for (int t = 0; t < HD / 16; t += 4) {
                        uint32_t f[4][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int ch = ((t + e) & 3) * 2 + ((lane >> 3) & 1);
                            ldsm4_t(f[e], rowa + (t >> 2) * col_ld + ((ch ^ (row & 7)) << 4));
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                mma16816<F16>(o[t + e][nt], f[e], pf[nt][0], pf[nt][1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                mma16816<F16>(o[t + e][nt], f[e], pl[nt][0], pl[nt][1]);
                    }
                }
                if (key0 < key_lo || key0 + 16 > key_hi) fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }

        // the four warps' sums, one after another in a fixed order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1)
                    l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
                if (lane < 4) {
                    wm[warp][nt * 8 + cq + e] = m[nt][e];
                    wl[warp][nt * 8 + cq + e] = l[nt][e];
                }
            }
        bar_sync(1, kWarps * 32);
        const bool uncut = p.k0 == 0 && p.k1 == p.nb;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt > 0) bar_sync(1, kWarps * 32);  // (the last rows have been read)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = nt * 8 + cq + e;
                const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
                const float f = m[nt][e] == -INFINITY ? 0.f : ex2((m[nt][e] - M) * cs);
                // [warp][row][dim], the dims swizzled so that neither side has bank conflicts
                float *dst = red + (warp * 8 + cq + e) * HD;
                const int sw = (cq >> 1) * 8;
#pragma unroll
                for (int t = 0; t < HD / 16; ++t) {
                    dst[(t * 16 + kr) ^ sw] = o[t][nt][e] * f;
                    dst[(t * 16 + 8 + kr) ^ sw] = o[t][nt][e + 2] * f;
                }
            }
            bar_sync(1, kWarps * 32);
            for (int i = threadIdx.x; i < HD; i += kWarps * 32) {  // 8 rows x HD / 8 pieces
                const int rr = i / (HD / 8), d0 = i % (HD / 8) * 8, r = nt * 8 + rr;
                if (r >= valid) continue;
                float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, L = 0.f;
                const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // (by the sum: a warp whose scores are all NaN has no maximum either)
                    L += wl[w][r] == 0.f ? 0.f : wl[w][r] * ex2((wm[w][r] - M) * cs);
                    const float *src = red + (w * 8 + rr) * HD + (d0 ^ (rr >> 1) * 8);
                    const float4 u = *reinterpret_cast<const float4 *>(src);
                    const float4 v = *reinterpret_cast<const float4 *>(src + 4);
                    y[0] += u.x;
                    y[1] += u.y;
                    y[2] += u.z;
                    y[3] += u.w;
                    y[4] += v.x;
                    y[5] += v.y;
                    y[6] += v.z;
                    y[7] += v.w;
                }
                if (uncut) {
                    const float f = L == 0.f ? 0.f : 1.f / L;
                    const uint4 v = make_uint4(
                        pack_t2<F16>(y[0] * f, y[1] * f), pack_t2<F16>(y[2] * f, y[3] * f),
                        pack_t2<F16>(y[4] * f, y[5] * f), pack_t2<F16>(y[6] * f, y[7] * f));
                    *reinterpret_cast<uint4 *>(a.out + (int64_t)(p.s.q0 + p.t0 + r / G) * a.out_ld +
                                               (int64_t)(p.h * G + r % G) * HD + d0) = v;
                } else {
                    const int64_t row = (int64_t)(2 * blockIdx.x + (p.k0 == 0 ? 1 : 0)) * kRows + r;
                    float4 *dst = reinterpret_cast<float4 *>(a.part_o + row * HD + d0);
                    dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                    dst[1] = make_float4(y[4], y[5], y[6], y[7]);
                    if (d0 == 0)
                        *reinterpret_cast<float2 *>(a.part_ml + row * 2) = make_float2(M * cs, L);
                }
            }
        }
        if (warp == 0) {
            if (p.parts > 0) {
                note_left = true;
                if (lane == 0)
                    a.notes[blockIdx.x] = SplitNote{p.s.q0 + p.t0, p.h * G, p.t1 - p.t0, p.parts};
            }
            if (lane == 0) stop = *abort;
        }
        bar_sync(1, kWarps * 32);
        if (stop) {  // one decision for all four warps
            // Given up: loads that nobody waits for any more end before this CTA does (they
            // take microseconds).  The loading warp's way out has no step for it: with a vote
            // or a wait there, one token over 200 keys took 7.5 us instead of 7.2.
            const unsigned long long t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 10000000ull) {
            }
            break;
        }
    }
    if (warp == 0 && lane == 0 && !note_left && !a.whole) a.notes[blockIdx.x] = SplitNote{0, 0, 0, 0};
}

// slot of part i of the tile that CTA c begins
__device__ __forceinline__ int64_t part_slot(int c, int i) {
    return i == 0 ? 2 * (int64_t)c + 1 : 2 * ((int64_t)c + i);
}

// Joins the parts of the tiles that several CTAs shared, in the CTAs' order:
// paged_rows_kernel's, [row][dim], few rows in many parts.  One CTA per row; its
// four warps take the parts in turn, once, with running maxima that they join at
// the end.
template <int HD, bool F16>
__global__ void __launch_bounds__(128) paged_merge_rows_kernel(const PagedAttnArgs a, int rows) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float sums[4][HD + 2];
    const SplitNote note = a.notes[blockIdx.x];
    const int G = a.n_heads / a.n_kv;
    if (!note_fits(note, blockIdx.x, gridDim.x, a.pb.n_tokens, a.n_heads, G)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = blockIdx.y;
    if (r >= note.tokens * G) return;
    constexpr int kPer = HD / 32, kAhead = 4;
    float M = -INFINITY, L = 0.f, acc[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
    for (int i0 = warp; i0 < note.parts; i0 += 4 * kAhead) {
        float2 ml[kAhead], v[kAhead][kPer / 2];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i0 + 4 * e >= note.parts) break;
            const int64_t at = part_slot(blockIdx.x, i0 + 4 * e) * rows + r;
            ml[e] = *reinterpret_cast<const float2 *>(a.part_ml + at * 2);
#pragma unroll
            for (int j = 0; j < kPer / 2; ++j)
                v[e][j] = *reinterpret_cast<const float2 *>(a.part_o + at * HD + lane * kPer + 2 * j);
        }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i0 + 4 * e >= note.parts || ml[e].y == 0.f) continue;
            const float mn = fmaxf(M, ml[e].x);
            const float f = M == -INFINITY ? 0.f : ex2(M - mn), g = ex2(ml[e].x - mn);
            M = mn;
            L = fmaf(L, f, ml[e].y * g);
#pragma unroll
            for (int j = 0; j < kPer / 2; ++j) {
                acc[2 * j] = fmaf(acc[2 * j], f, v[e][j].x * g);
                acc[2 * j + 1] = fmaf(acc[2 * j + 1], f, v[e][j].y * g);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) sums[warp][lane * kPer + j] = acc[j];
    if (lane == 0) {
        sums[warp][HD] = L;
        sums[warp][HD + 1] = M;
    }
    __syncthreads();
    if (warp > 0) return;
    M = fmaxf(fmaxf(sums[0][HD + 1], sums[1][HD + 1]), fmaxf(sums[2][HD + 1], sums[3][HD + 1]));
    L = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = sums[w][HD] == 0.f ? 0.f : ex2(sums[w][HD + 1] - M);
        L = fmaf(sums[w][HD], f, L);
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[j] = fmaf(sums[w][lane * kPer + j], f, acc[j]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t *op = a.out + (int64_t)(note.q_row + r / G) * a.out_ld +
                   (int64_t)(note.heads0 + r % G) * HD + lane * kPer;
#pragma unroll
    for (int j = 0; j < kPer; j += 2)
        *reinterpret_cast<uint32_t *>(op + j) = pack_t2<F16>(acc[j] * inv, acc[j + 1] * inv);
}

// The same for paged_tiles_kernel's parts, [dim / 4][row][4] (its threads have a
// row each), many rows in few parts: one thread takes 8 dims of a row, so that
// a warp reads 512 bytes in one piece, and goes through the parts once with a
// running maximum, four parts' loads under way.
template <int HD, bool F16>
__global__ void __launch_bounds__(128) paged_merge_tiles_kernel(const PagedAttnArgs a, int rows) {
    pdl_launch_dependents();
    pdl_wait();
    const SplitNote note = a.notes[blockIdx.x];
    const int G = a.n_heads / a.n_kv;
    if (!note_fits(note, blockIdx.x, gridDim.x, a.pb.n_tokens, a.n_heads, G)) return;
    const int r = blockIdx.z * 128 + threadIdx.x, d0 = blockIdx.y * 8;
    if (r >= note.tokens * G) return;
    float M = -INFINITY, L = 0.f, acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    constexpr int kAhead = 4;
    for (int i0 = 0; i0 < note.parts; i0 += kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead][2];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i0 + e >= note.parts) break;
            const int64_t at = part_slot(blockIdx.x, i0 + e) * rows;
            ml[e] = *reinterpret_cast<const float2 *>(a.part_ml + (at + r) * 2);
            const float *po = a.part_o + at * HD + ((d0 >> 2) * rows + r) * 4;
#pragma unroll
            for (int j = 0; j < 2; ++j) v[e][j] = *reinterpret_cast<const float4 *>(po + j * rows * 4);
        }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            if (i0 + e >= note.parts || ml[e].y == 0.f) continue;
            const float mn = fmaxf(M, ml[e].x);
            const float f = M == -INFINITY ? 0.f : ex2(M - mn), g = ex2(ml[e].x - mn);
            M = mn;
            L = fmaf(L, f, ml[e].y * g);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[4 * j] = fmaf(acc[4 * j], f, v[e][j].x * g);
                acc[4 * j + 1] = fmaf(acc[4 * j + 1], f, v[e][j].y * g);
                acc[4 * j + 2] = fmaf(acc[4 * j + 2], f, v[e][j].z * g);
                acc[4 * j + 3] = fmaf(acc[4 * j + 3], f, v[e][j].w * g);
            }
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint4 *>(a.out + (int64_t)(note.q_row + r / G) * a.out_ld +
                               (int64_t)(note.heads0 + r % G) * HD + d0) =
        make_uint4(pack_t2<F16>(acc[0] * inv, acc[1] * inv), pack_t2<F16>(acc[2] * inv, acc[3] * inv),
                   pack_t2<F16>(acc[4] * inv, acc[5] * inv), pack_t2<F16>(acc[6] * inv, acc[7] * inv));
}

// CTAs of paged_rows_kernel: as many as fit at once
int rows_grid(int hd) {
    return sm_count() *
           (hd == 64 ? Cfg<64>::kCtas : (hd == 128 ? Cfg<128>::kCtas : Cfg<256>::kCtas));
}

// Which kernel serves a call: paged_rows_kernel while a sequence's new tokens
// make one tile of 16 rows, so that each key is read once; the tensor-core
// kernel (128- or 256-row tiles) from there on.
// Tiles are left whole where no sequence, or no window with a tile's tokens, can
// have more than kWholeKeys (kWholeKeysTiles) keys, by the table's width: a few
// blocks take less than the parts and their merge.  Cut -> whole, us: one token
// over 256 keys 8.7 -> 7.3, over 512 8.7 -> 10.5; a windowed chunk (1024 keys)
// 45.6 -> 35.2; prompts of 512 / 1024 / 1280 tokens, 32 heads of 8 key heads, 26.5 ->
// 18.2, 37.7 -> 26.4, 43.5 -> 37.3 (but 4 heads of one key head, a few tiles on 148
// SMs, 18.9 -> 17.1, 20.5 -> 24.3, 21.4 -> 27.9).  Where the tiles are as many as the
// SMs, twice as many keys (a prompt of 2048 62.0 -> 50.8; 2560 81 -> 94).
struct Shape {
    bool tiles, whole;
    int grid, rows, block;  // CTAs, rows of a part, keys of a block
};

constexpr int64_t kWholeKeys = 256, kWholeKeysTiles = 1280;

Shape shape_of(int n_heads, int n_kv, int hd, int64_t max_q, int64_t max_keys, int64_t n_tokens,
               int64_t window) {
    const int G = n_heads / n_kv;
    if (max_q > kRows / G) {
        const int rows = paged_tiles_rows(hd), TT = rows / 128 * (128 / G);
        const int64_t span = window > 0 ? std::min(max_keys, window + TT) : max_keys;
        const bool many = n_tokens / TT * n_kv >= sm_count();
        return Shape{true, span <= kWholeKeysTiles * (many ? 2 : 1), sm_count(), rows, 128};
    }
    return Shape{false, max_keys <= kWholeKeys, rows_grid(hd), kRows, kBlock};
}

template <int HD, bool F16, int NT>
cudaError_t run_rows(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                     cudaStream_t st) {
    auto kern = paged_rows_kernel<HD, F16, NT>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, Cfg<HD>::kSmem, allowed);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3((unsigned)rows_grid(HD)), kThreads, Cfg<HD>::kSmem, st, mk, mv, a);
}

template <int HD, bool F16>
cudaError_t run_attention(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                          const Shape &s, int64_t rows, cudaStream_t st) {
    const cudaError_t e = s.tiles     ? launch_paged_tiles(a, mk, mv, HD, F16, st)
                          : rows <= 8 ? run_rows<HD, F16, 1>(a, mk, mv, st)
                                      : run_rows<HD, F16, 2>(a, mk, mv, st);
    if (e != cudaSuccess || s.whole) return e;
    if (s.tiles)
        return launch_pdl(paged_merge_tiles_kernel<HD, F16>,
                          dim3((unsigned)s.grid, HD / 8, (unsigned)s.rows / 128), 128, 0, st, a,
                          s.rows);
    // (a caller's max_q may be too small: every row of a tile has its CTA)
    return launch_pdl(paged_merge_rows_kernel<HD, F16>, dim3((unsigned)s.grid, rows <= 8 ? 8u : 16u),
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
    auto bytes = [&](int64_t q) {
        const Shape s = shape_of(n_heads, n_kv, head_dim, q, max_keys, 0, 0);
        return s.whole ? 0 : part_bytes(s.grid, s.rows, head_dim);
    };
    return max_q > 0 ? bytes(max_q) : std::max(bytes(1), bytes(kRows + 1));  // (0: any)
}

cudaError_t launch_paged_attention(const PagedAttnCall &c, cudaStream_t st) {
    const Shape s = shape_of(c.n_heads, c.n_kv, c.head_dim, c.max_q,
                             (int64_t)c.pb.table_width * c.pb.page_size, c.pb.n_tokens, c.window);
    // (of the rows kernel, which has at most kRows)
    const int64_t rows = std::min<int64_t>(c.max_q, kRows) * (c.n_heads / c.n_kv);
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
    a.whole = s.whole;
    // the largest power of two that divides the page size: no box crosses a page
    a.box = std::min(s.block, c.pb.page_size & -c.pb.page_size);
    // (the tensor-core kernel's stages hold 128 dims, its columns 128 keys)
    a.box_cols = !s.tiles ? c.head_dim / 64 : (a.box == s.block && c.head_dim > 64 ? 2 : 1);
    if (!s.whole) place_workspace(a, s.grid, s.rows, c.ws);
    CUtensorMap mk, mv;
    if (!make_map_pages(&mk, c.f16, c.k, c.head_dim, c.pb.page_size, c.n_kv, c.pb.n_pages,
                        c.page_stride, a.box, a.box_cols) ||
        !make_map_pages(&mv, c.f16, c.v, c.head_dim, c.pb.page_size, c.n_kv, c.pb.n_pages,
                        c.page_stride, a.box, a.box_cols))
        return cudaErrorInvalidValue;
    if (c.f16) {
        if (c.head_dim == 64) return run_attention<64, true>(a, mk, mv, s, rows, st);
        if (c.head_dim == 128) return run_attention<128, true>(a, mk, mv, s, rows, st);
        return run_attention<256, true>(a, mk, mv, s, rows, st);
    }
    if (c.head_dim == 64) return run_attention<64, false>(a, mk, mv, s, rows, st);
    if (c.head_dim == 128) return run_attention<128, false>(a, mk, mv, s, rows, st);
    return run_attention<256, false>(a, mk, mv, s, rows, st);
}

}  // namespace nq
