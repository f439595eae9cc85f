// attn_paged_tc.cu -- attention of new tokens over the paged cache for many
// query rows per key head (chunks of a prompt), on tcgen05 tensor cores.  The
// mathematics and the split over the CTAs are attn_paged.cu's; paged.cuh has
// the split.
//
// A query tile is 128 rows (the G query heads of a key head times 128 / G
// tokens), a key block 128 keys.  One CTA per SM, persistent over its pieces:
//   key and value warp   K and V blocks into a ring of stages each by TMA (128-byte
//                 swizzle, boxes of 16 to 128 keys x 64 dims; a warp starts a box
//                 about every 65 ns, so small pages ask for two warps)
//   MMA warp      S = Q K^T (both in shared memory) and O += P V (P in TMEM, V as
//                 it lies: keys x dims, the MN-major operand), one thread
//   query warp    the next tile's queries, as soon as the last S that reads the
//                 present ones is done
//   softmax       one row per thread: S from TMEM, a running maximum and sum,
//                 P back into S's columns in 16 bits
// Two tiles S are always in flight, so that the tensor cores work on one while
// the softmax warps work on the other:
//   two query tiles  (more than 128 / G tokens): one warpgroup each, and each
//                    key block is read once for 256 rows
//   one query tile   two warpgroups take the key blocks in turn, each with a
//                    maximum, sum and O of its own, joined at the end
//   256 dims         O fills half of the TMEM: one warpgroup, one O, two S
// O is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time; until then the weights are up to 2^8, which costs neither bf16
// nor fp16 precision.
//
// A prompt of 8192 tokens (32 heads of 128 dims, 550 GFLOP): 485 us, 1.13 PFLOP/s,
// in a short run, 560 us where the power limit holds the clock at 1.4 GHz.  What
// bounds it is the chain of a group's S: about 2000 cycles of softmax (128 * 128
// exponentials on the SM's 16 a cycle take 1024 of them) and 1450 from the last
// weight to the next S, with the other group's products in between.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "nq_common.cuh"
#include "nq_internal.h"
#include "paged.cuh"

namespace nq {
namespace {

constexpr int kBlock = 128;  // keys per block, rows per query tile

template <int HD>
struct Tc {
    static constexpr int kGroups = HD == 256 ? 1 : 2;       // softmax warpgroups
    static constexpr int kMmaWarp = 4 * kGroups, kKeyWarp = kMmaWarp + 1;
    static constexpr int kValueWarp = kKeyWarp + 1, kQueryWarp = kValueWarp + 1;
    // The last warpgroup is one MMA, one key, one value and one query warp.  With
    // two softmax warpgroups registers are moved between them: 168 each at launch
    // (all of the SM's 64 K), then 208 for a softmax thread, which holds a row of 128
    // scores, and 88 for the others; 2 * 208 + 88 = 3 * 168.
    static constexpr int kThreads = 128 * (kGroups + 1);
    // S in TMEM per group, beside O.  One each for two groups: 64 keys in two S each
    // would have the next S ready when a softmax is done, but an MMA of 64 columns
    // takes 68 cycles where one of 128 takes 83 (its 128 query rows come from shared
    // memory either way), and a prompt of 8192 tokens 556 us instead of 496.
    static constexpr int kBufs = kGroups == 2 ? 1 : 2;
    // The weights of a step's first kMost keys are handed over early, so that most of
    // P V runs while the rest are still being made (96 of 128: a prompt of 8192 tokens
    // 519 -> 492 us; with 256 dims, where the MMAs are the bound, 440 -> 475).
    static constexpr int kMost = kGroups == 2 ? 96 : kBlock;
    // a ring stage: 128 keys (or values) x kUnitDims dims
    static constexpr int kUnitDims = HD < 128 ? HD : 128;
    static constexpr int kUnits = HD / kUnitDims;
    static constexpr int kUnitBytes = kBlock * kUnitDims * 2;
    static constexpr int kStages = HD == 64 ? 4 : 2;  // of keys, and as many of values: 128 KB
    static constexpr int kQBytes = kBlock * HD * 2;
    static constexpr int kOutBytes = 2048;                  // a warp's 32 rows x 32 dims
    static constexpr int kSmem =
        kGroups * kQBytes + 2 * kStages * kUnitBytes + 4 * kGroups * kOutBytes;
    static constexpr int kO = 256;                          // first TMEM column of O
    static constexpr int kRows = kGroups * kBlock;          // rows of a part
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 values per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Named barrier over `count` threads; whether any of them said so.
__device__ __forceinline__ bool bar_any(int id, int count, bool x) {
    int y;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(y)
        : "r"((int)x), "r"(id), "r"(count)
        : "memory");
    return y != 0;
}

// mbar_wait_or_abort() for the hand-overs between the MMA and softmax warps,
// which happen every microsecond: a thread that suspends in try_wait wakes up
// to 300 cycles after the last arrival, one that polls within 50.
__device__ __forceinline__ bool mbar_poll_or_abort(uint64_t *bar, uint32_t parity,
                                                   volatile int *abort, unsigned int *err) {
    unsigned long long t0 = 0;
    for (int i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 255) != 255) continue;
        if (*abort) return false;
        if (t0 == 0) t0 = global_timer_ns();
        if (global_timer_ns() - t0 > kWaitLimitNs) {
            *abort = 1;
            atomicOr(err, kErrWaitTimeout);
            return false;
        }
    }
}

// MMAs and commits run by a whole warp, one lane of which issues.  Under a
// branch on the lane every operand of every MMA would be moved from vector to
// uniform registers first, about 100 cycles for an MMA that takes 64; with
// warp-uniform operands they stay in uniform registers.
// D[tmem] (+)= A[smem] * B[smem]^T, kind::f16; the descriptors' upper halves are
// constants.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                       uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\telect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 y;\n\telect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            smem_u32(bar))
        : "memory");
}

// The lower half of a descriptor of an operand at 1024-byte aligned smem_addr,
// and the upper halves (128-byte swizzle, stride offset 1024 bytes).  K along
// memory: smem_desc_k_sw128().  N (here: dims) along memory: atoms of 64 dims x 8
// keys, the next 8 keys 1024 bytes on (stride offset), the next 64 dims a
// 128-key column of 16 KB on (leading offset).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t smem_addr) {
    return ((smem_addr >> 4) & 0x3FFFu) | (1u << 16);
}
__device__ __forceinline__ uint32_t desc_mn(uint32_t smem_addr) {
    return ((smem_addr >> 4) & 0x3FFFu) | ((16384u >> 4) << 16);
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]));
}

// The blocks of a piece as the groups' steps; step i works on the group's S
// buffer i % kBufs.
template <int HD>
struct Plan {
    bool two;    // two query tiles, a group each; else the groups take the blocks in turn
    int n;       // blocks
    __device__ __forceinline__ Plan(const Piece &p, int tok)
        : two(Tc<HD>::kGroups == 2 && p.t1 - p.t0 > tok), n(p.k1 - p.k0) {}
    __device__ __forceinline__ bool turns() const { return Tc<HD>::kGroups == 2 && !two; }
    __device__ __forceinline__ int steps(int w) const { return turns() ? (n + 1 - w) / 2 : n; }
    __device__ __forceinline__ int block(int w, int i) const { return turns() ? 2 * i + w : i; }
    // whether group w is the last that uses a block's keys and values
    __device__ __forceinline__ bool last_use(int w) const { return !two || w == 1; }
};

// A piece as the key warp, which alone walks the list, hands it to the others
// (two slots, so that it runs a piece ahead); n: its blocks, 0 at the list's end.
struct Job {
    Piece p;
    int n;
};

// Where a lane's box of a key block lies: its page (n_pages, whose reads give
// zeros, for a box without a visible key of the piece) and row in the page.
struct Place {
    int page, slot;
};
__device__ __forceinline__ Place box_place(const PagedAttnArgs &a, int row, int key, bool on,
                                           int key_lo, int key_hi) {
    Place p{a.pb.n_pages, 0};
    if (on && key < key_hi && key + a.box > key_lo) {
        p.page = page_of(a.pb, row, key);
        p.slot = key % a.pb.page_size;
    }
    return p;
}

template <int HD, bool F16>
__global__ void __launch_bounds__(Tc<HD>::kThreads, 1) paged_tiles_kernel(
    const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
    const __grid_constant__ CUtensorMap mv, const PagedAttnArgs a) {
    using T = Tc<HD>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *qs = smem, *ring_k = smem + T::kGroups * T::kQBytes;
    uint8_t *ring_v = ring_k + T::kStages * T::kUnitBytes;
    uint8_t *outs = ring_v + T::kStages * T::kUnitBytes;
    // a ring of keys and one of values: a ring has one producer, or its waits would be
    // ambiguous
    __shared__ __align__(8) uint64_t full_k[T::kStages], empty_k[T::kStages];
    __shared__ __align__(8) uint64_t full_v[T::kStages], empty_v[T::kStages];
    __shared__ __align__(8) uint64_t s_full[2], p_most[2], p_ready[2];  // per S
    __shared__ __align__(8) uint64_t q_full, q_empty, o_full, pv_done[T::kGroups];
    __shared__ uint32_t tmem_holder;
    __shared__ int abort_flag;
    __shared__ float2 xml[T::kGroups == 2 ? 2 * kBlock : 1];
    __shared__ Job jobs[2];
    __shared__ __align__(8) uint64_t job_full[2], job_empty[2];
    volatile int *abort = &abort_flag;
    // (the shuffle tells the compiler that the roles' branches are warp-uniform)
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const int G = a.n_heads / a.n_kv, tok = kBlock / G, TT = T::kGroups * tok;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < T::kStages; ++i) {
            mbar_init(&full_k[i], 1);
            mbar_init(&empty_k[i], 1);
            mbar_init(&full_v[i], 1);
            mbar_init(&empty_v[i], 1);
        }
        for (int i = 0; i < T::kGroups; ++i) mbar_init(&pv_done[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_most[i], 4);  // (one arrival per warp)
            mbar_init(&p_ready[i], 4);
            mbar_init(&job_full[i], 1);
            mbar_init(&job_empty[i], 3 + 4 * T::kGroups);  // the other warps
        }
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        mbar_init(&o_full, 1);
        abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&mq);
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    if (warp == T::kMmaWarp) {
        tmem_alloc(&tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    pdl_wait();  // lengths, tables, q and the cache come from earlier kernels

    if (warp >= 4 * T::kGroups) {
    if constexpr (T::kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // K and V of a block: kUnitDims dims per ring stage, as columns of 64 dims (16 KB
    // each), in boxes of a.box keys, a lane each; a box of all 128 keys takes both
    // columns.  The pages of the next block are looked up ahead.
    auto load = [&](const Piece &p, const CUtensorMap *map, uint8_t *ring, uint64_t *full,
                    uint64_t *empty, int &g) {
        constexpr int kCols = T::kUnitDims / 64;
        const int per = kCols / a.box_cols, box_r = lane / per, box_c = lane % per;
        const bool on = box_r < kBlock / a.box;
        const uint32_t box_at = box_c * (kBlock * 128) + box_r * a.box * 128;
        const int n = p.k1 - p.k0;
        const int p0 = p.s.len - p.s.n + p.t0, key_hi = p.s.len - p.s.n + p.t1;
        const int key_lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
        const int key0 = (p.lo + p.k0) * kBlock + box_r * a.box;
        Place next = box_place(a, p.s.row, key0, on, key_lo, key_hi);
        for (int b = 0; b < n; ++b) {
            const Place at = next;
            next = box_place(a, p.s.row, key0 + (b + 1) * kBlock, on && b + 1 < n, key_lo, key_hi);
#pragma unroll
            for (int u = 0; u < T::kUnits; ++u, ++g) {
                const int st = g % T::kStages;
                if (!warp_wait_or_abort(&empty[st], (uint32_t)(g / T::kStages + 1) & 1u, abort,
                                        a.pb.err))
                    return false;
                if (lane == 0) mbar_expect_tx(&full[st], T::kUnitBytes);
                __syncwarp();
                if (on)
                    tma_load_5d(ring + st * T::kUnitBytes + box_at, map, &full[st], 0, at.slot,
                                u * kCols + box_c, p.h, at.page);
            }
        }
        return true;
    };
    if (warp == T::kKeyWarp) {
        const Tiling tl{TT, T::kGroups == 2 ? tok : TT, a.window, a.whole};
        Share sh = find_share<kBlock>(a.pb, a.n_kv, tl, blockIdx.x, gridDim.x);
        Piece p;
        int filled = 0, jobs_out = 0;
        bool ok = true;
        // no tile of this CTA's is cut, until a softmax thread says so (which it does
        // behind a job, and not where it has given up: the merge always finds a note)
        if (lane == 0 && !a.whole) a.notes[blockIdx.x] = SplitNote{0, 0, 0, 0};
        auto hand_out = [&](int n) {
            const int slot = jobs_out & 1;
            ok = warp_wait_or_abort(&job_empty[slot], (uint32_t)(jobs_out / 2 + 1) & 1u, abort,
                                    a.pb.err);
            if (ok && lane == 0) {
                jobs[slot].p = p;
                jobs[slot].n = n;
                mbar_arrive(&job_full[slot]);
            }
            ++jobs_out;
        };
        while (ok && next_piece<kBlock>(a.pb, a.n_kv, tl, sh, blockIdx.x, p)) {
            hand_out(p.k1 - p.k0);
            ok = ok && load(p, &mk, ring_k, full_k, empty_k, filled);
        }
        if (ok) hand_out(0);
    } else if (warp == T::kValueWarp) {
        int filled = 0;
        for (int pieces = 0;; ++pieces) {
            const int slot = pieces & 1;
            if (!warp_wait_or_abort(&job_full[slot], (uint32_t)(pieces / 2) & 1u, abort, a.pb.err) ||
                jobs[slot].n == 0)
                break;
            const Piece p = jobs[slot].p;
            __syncwarp();
            if (lane == 0) mbar_arrive(&job_empty[slot]);
            if (!load(p, &mv, ring_v, full_v, empty_v, filled)) break;
        }
    } else if (warp == T::kMmaWarp) {
        constexpr uint32_t kIdS = F16 ? idesc_f16_f32(128, 128) : idesc_bf16_f32(128, 128);
        constexpr uint32_t kIdO = (F16 ? idesc_f16_f32(128, T::kUnitDims)
                                       : idesc_bf16_f32(128, T::kUnitDims)) |
                                  (1u << 16);  // B: N along memory
        const uint32_t q_lo = desc_k(smem_u32(qs)), k_lo = desc_k(smem_u32(ring_k)),
                       v_lo = desc_mn(smem_u32(ring_v));
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        int blocks = 0, pieces = 0;  // finished
        uint32_t p_phase = 0;        // bit: parity of that S's next p_most and p_ready
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_poll_or_abort(bar, parity, abort, a.pb.err)) != 0;
        };
        auto wait_stage = [&](uint64_t *full, int g) {
            ok = ok && wait(&full[g % T::kStages], (uint32_t)(g / T::kStages) & 1u);
        };
        while (ok) {
            const int slot = pieces & 1;
            ok = wait(&job_full[slot], (uint32_t)(pieces / 2) & 1u);
            if (!ok) break;
            Plan<HD> pl(jobs[slot].p, tok);
            pl.n = __shfl_sync(0xffffffffu, jobs[slot].n, 0);
            pl.two = __all_sync(0xffffffffu, pl.two);
            if (pl.n == 0) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&job_empty[slot]);
            ok = wait(&q_full, (uint32_t)pieces & 1u);
            int s_left = T::kGroups == 2 ? pl.steps(0) + pl.steps(1) : pl.steps(0);
            auto issue_s = [&](int w, int i) {
                const int b = pl.block(w, i), at = w * T::kBufs + i % T::kBufs;
                const uint32_t qd = q_lo + (pl.two && w ? T::kQBytes >> 4 : 0);
#pragma unroll
                for (int u = 0; u < T::kUnits; ++u) {
                    const int g = (blocks + b) * T::kUnits + u;
                    wait_stage(full_k, g);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t kd = k_lo + (g % T::kStages) * (T::kUnitBytes >> 4);
#pragma unroll
                    for (int kk = 0; kk < T::kUnitDims / 16; ++kk) {
                        // 16 dims: 32 bytes on in the swizzled rows; 64: the next column
                        const uint32_t off = ((kk >> 2) * (kBlock * 128) + (kk & 3) * 32) >> 4;
                        mma_ss(tm + at * kBlock,
                               qd + (u * (T::kUnitDims / 64) * (kBlock * 128) >> 4) + off, kDescHi,
                               kd + off, kDescHi, kIdS, (u > 0 || kk > 0) ? 1u : 0u);
                    }
                    if (pl.last_use(w)) mma_commit(&empty_k[g % T::kStages]);
                }
                mma_commit(&s_full[at]);
                if (--s_left == 0) mma_commit(&q_empty);
            };
#pragma unroll
            for (int i = 0; i < T::kBufs; ++i)
#pragma unroll
                for (int w = 0; w < T::kGroups; ++w)
                    if (ok && i < pl.steps(w)) issue_s(w, i);
            for (int i = 0; ok && i < pl.steps(0); ++i) {
                // (not unrolled: all roles' code shares one instruction cache, and two copies
                // of this one cost a prompt of 8192 tokens 532 us instead of 483)
#pragma unroll 1
                for (int w = 0; w < T::kGroups; ++w) {
                    if (i >= pl.steps(w)) continue;
                    const int b = pl.block(w, i), at = w * T::kBufs + i % T::kBufs;
                    ok = ok && wait(T::kMost < kBlock ? &p_most[at] : &p_ready[at],
                                    (p_phase >> at) & 1u);
                    if (!ok) break;
                    const uint32_t o = tm + T::kO + w * HD;
#pragma unroll
                    for (int u = 0; u < T::kUnits; ++u) {
                        const int g = (blocks + b) * T::kUnits + u;
                        wait_stage(full_v, g);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t vd = v_lo + (g % T::kStages) * (T::kUnitBytes >> 4);
#pragma unroll
                        for (int kk = 0; kk < kBlock / 16; ++kk) {
                            if (u == 0 && kk == T::kMost / 16) {
                                ok = wait(&p_ready[at], (p_phase >> at) & 1u);
                                if (!ok) break;
                                tc_fence_after();
                            }
                            mma_ts(o + u * T::kUnitDims, tm + at * kBlock + kk * 8,
                                   vd + (kk * 16 * 128 >> 4), kDescHi, kIdO,
                                   (i > 0 || kk > 0) ? 1u : 0u);
                        }
                        if (!ok) break;
                        if (pl.last_use(w)) mma_commit(&empty_v[g % T::kStages]);
                    }
                    p_phase ^= 1u << at;
                    mma_commit(&pv_done[w]);
                    if (ok && i + T::kBufs < pl.steps(w)) issue_s(w, i + T::kBufs);
                }
            }
            mma_commit(&o_full);
            blocks += pl.n;
            ++pieces;
        }
        if (!ok && pieces > 0) {  // given up: the products in flight end first
            const unsigned long long t0 = global_timer_ns();
            while (!mbar_try_wait(&o_full, (uint32_t)(pieces - 1) & 1u) &&
                   global_timer_ns() - t0 < kWaitLimitNs) {
            }
        }
        __syncwarp();
    } else if (warp == T::kQueryWarp) {
        // ---------------------------------------------------------- query rows
        // G heads of tok tokens are a tile's rows in their order; the rows of a tile's
        // missing tokens hold another sequence's, or zeros: their scores are masked.
        for (int pieces = 0; lane == 0; ++pieces) {
            const int slot = pieces & 1;
            if (!mbar_wait_or_abort(&job_full[slot], (uint32_t)(pieces / 2) & 1u, abort, a.pb.err) ||
                jobs[slot].n == 0)
                break;
            const int row = jobs[slot].p.s.q0 + jobs[slot].p.t0, h = jobs[slot].p.h * G;
            const int subs = Plan<HD>(jobs[slot].p, tok).two ? 2 : 1;
            mbar_arrive(&job_empty[slot]);
            if (!mbar_wait_or_abort(&q_empty, (uint32_t)(pieces + 1) & 1u, abort, a.pb.err)) break;
            mbar_expect_tx(&q_full, subs * (HD / 64) * tok * G * 128);
            for (int sub = 0; sub < subs; ++sub)
                for (int col = 0; col < HD / 64; ++col)
                    tma_load_4d(qs + sub * T::kQBytes + col * (kBlock * 128), &mq, &q_full, 0, h,
                                row + sub * tok, col);
        }
        __syncwarp();
    }
    } else {
        // ---------------------------------------------------------- softmax
        if constexpr (T::kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int w = warp >> 2;                    // warpgroup
        const int r = threadIdx.x & 127;            // this thread's row of the query tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float cs = a.scale * 1.4426950408889634f;  // exp(scale x) = 2^(cs x)
        const uint32_t inv_g = (65535 + G) / G;  // r / G = r * inv_g >> 16 for r < 128
        int blocks = 0, pieces = 0, pvs = 0;
        uint32_t s_phase = 0;
        bool ok = true;
        while (true) {
            // What a piece says stays in shared memory until it is needed: the scores take
            // most of the registers.
            const Job &job = jobs[pieces & 1];
            ok = ok && !*abort &&
                 mbar_wait_or_abort(&job_full[pieces & 1], (uint32_t)(pieces / 2) & 1u, abort,
                                    a.pb.err);
            // (one decision for both warpgroups: each takes part in the barrier below, or
            // neither does)
            if (T::kGroups == 2)
                ok = !bar_any(1, 256, !ok);
            else
                ok = __all_sync(0xffffffffu, ok);
            if (!ok || job.n == 0) break;
            const Piece &p = job.p;
            const Plan<HD> pl(p, tok);
            const int steps = pl.steps(w);
            const int sub = pl.two ? w : 0;         // which query tile
            const int t0 = p.t0 + sub * tok, t1 = min(t0 + tok, p.t1);
            const int valid = (t1 - t0) * G;
            const int base = p.s.len - p.s.n;
            const int pos = r < valid ? base + t0 + (int)((uint32_t)r * inv_g >> 16) : -1;
            // steps whose keys reach past the first row's position, or below the last
            // row's window, are masked
            const int full_to = base + t0 + 1 - kBlock;
            const int full_from = a.window > 0 ? base + t1 - a.window : 0;
            const int block0 = p.lo + p.k0;
            float m = -INFINITY, l = 0.f;
            for (int i = 0; i < steps; ++i) {
                const int buf = i % T::kBufs, at = w * T::kBufs + buf, b = pl.block(w, i);
                ok = ok && !*abort &&
                     mbar_poll_or_abort(&s_full[at], (s_phase >> buf) & 1u, abort, a.pb.err);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                s_phase ^= 1u << buf;
                tc_fence_after();
                const uint32_t sc = tmem + lanes + at * kBlock;
                float s[kBlock];
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                const int key0 = (block0 + b) * kBlock;
                const bool masked = key0 > full_to || key0 < full_from;
                const int hi = pos - key0, lo = a.window > 0 ? hi - a.window + 1 : 0;
                // (the second half on its way while the first one's maximum is taken)
                tmem_ld_32x32b_x32(sc, *reinterpret_cast<uint32_t(*)[32]>(s));
                tmem_ld_32x32b_x32(sc + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                tmem_ld_wait();
                tmem_ld_32x32b_x32(sc + 64, *reinterpret_cast<uint32_t(*)[32]>(s + 64));
                tmem_ld_32x32b_x32(sc + 96, *reinterpret_cast<uint32_t(*)[32]>(s + 96));
#pragma unroll
                for (int c = 0; c < kBlock; c += 64) {
                    if (c > 0) tmem_ld_wait();
                    if (masked) {
#pragma unroll
                        for (int j = c; j < c + 64; ++j)
                            if (j > hi || j < lo) s[j] = -INFINITY;
                    }
#pragma unroll
                    for (int j = c; j < c + 64; j += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x[e] = fmaxf(x[e], fmaxf(s[j + e], s[j + 4 + e]));
                }
                const float mn = fmaxf(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
                // (m == -inf: the difference is +inf, or NaN when the row has no key yet; rows
                // behind the tile's own, which the last tile may have left in shared memory,
                // have no say, or the rounding of this warp's other rows would follow them)
                if (__any_sync(0xffffffffu, r < valid && (mn - m) * cs > 8.f)) {
                    const float f = m == -INFINITY ? 0.f : ex2((m - mn) * cs);
                    if (i > 0) {
                        // O still takes the last step's product: wait for it
                        ok = mbar_wait_or_abort(&pv_done[w], (uint32_t)(pvs + i - 1) & 1u, abort,
                                                a.pb.err);
                        ok = __all_sync(0xffffffffu, ok);
                        tc_fence_after();
                        const uint32_t oc = tmem + lanes + T::kO + w * HD;
#pragma unroll 1
                        for (int j = 0; j < HD; j += 32) {
                            uint32_t v[32];
                            tmem_ld_32x32b_x32(oc + j, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                            tmem_st_32x32b_x32(oc + j, v);
                        }
                    }
                    l *= f;
                    m = mn;
                }
                const int key_hi = p.s.len - p.s.n + p.t1;
                const int key_lo = a.window > 0 ? p.s.len - p.s.n + p.t0 - a.window + 1 : 0;
                if (key0 < key_lo || key0 + kBlock > key_hi) {
                    // values of keys that no row sees may hold anything: a NaN times a
                    // weight of 0 would reach the sum
                    const int key = key0 + r;
                    const bool clear = (!pl.two || w == 0) && (key < key_lo || key >= key_hi);
                    // (256 dims: the stage's last values may still be under way, and a wait two
                    // phases ahead would be ambiguous)
                    if (T::kGroups == 1 && i > 0)
                        ok = ok && mbar_wait_or_abort(&pv_done[w], (uint32_t)(pvs + i - 1) & 1u,
                                                      abort, a.pb.err);
#pragma unroll
                    for (int u = 0; u < T::kUnits; ++u) {
                        const int g = (blocks + b) * T::kUnits + u;
                        ok = ok && mbar_wait_or_abort(&full_v[g % T::kStages],
                                                      (uint32_t)(g / T::kStages) & 1u, abort,
                                                      a.pb.err);
                        if (ok && clear) {
                            uint8_t *v = ring_v + (g % T::kStages) * T::kUnitBytes +
                                         r * 128;
#pragma unroll
                            for (int j = 0; j < T::kUnitDims / 8; ++j)
                                *reinterpret_cast<uint4 *>(v + (j >> 3) * (kBlock * 128) +
                                                           (j & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                const float z = m == -INFINITY ? 0.f : m * cs;
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int j = 0; j < kBlock / 32; ++j) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 x2 = fma2(make_float2(s[j * 32 + 2 * e], s[j * 32 + 2 * e + 1]),
                                               make_float2(cs, cs), make_float2(-z, -z));
                        const float e0 = ex2(x2.x), e1 = ex2(x2.y);
                        sum[e & 1] = add2(sum[e & 1], make_float2(e0, e1));
                        // Rounded to the cache's type: both factors of an MMA are of one type.
                        // (A second term, as attn_paged.cu's kernel takes, is as many MMAs and
                        // stores again on the chain that bounds this one: a prompt of 8192
                        // tokens 559 -> 754 us, for an error against 64 bits of 0.0017 instead
                        // of 0.0023; the result's own rounding makes 0.0017.)
                        pk[e] = pack_t2<F16>(e0, e1);
                    }
                    tmem_st_32x32b_x16(sc + j * 16, pk);
                    if (T::kMost < kBlock && j * 32 + 32 == T::kMost) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_most[at]);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[at]);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            ok = ok && !*abort &&
                 mbar_wait_or_abort(&o_full, (uint32_t)pieces & 1u, abort, a.pb.err);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const bool whole = p.k0 == 0 && p.k1 == p.nb;
            // One query tile in two warpgroups' sums: each thread can read its row of both
            // O, so a warpgroup writes half of the dims, joining the two as it goes.
            const bool join = T::kGroups == 2 && !pl.two;
            float f0 = 1.f, f1 = 0.f, M = m, L = l;
            if (join) {
                xml[w * kBlock + r] = make_float2(m, l);
                bar_sync(1, 256);
                const float2 a0 = xml[r], a1 = xml[kBlock + r];
                M = fmaxf(a0.x, a1.x);
                f0 = a0.x == -INFINITY ? 0.f : ex2((a0.x - M) * cs);
                f1 = a1.x == -INFINITY ? 0.f : ex2((a1.x - M) * cs);
                L = a0.y * f0 + a1.y * f1;
            }
            if (ok) {
                // (a row without a key: whatever O holds)
                const float inv = L == 0.f ? 0.f : (whole ? 1.f / L : 1.f);
                f0 *= inv;
                f1 *= inv;
                const bool both = join && pl.n > 1;  // (else the second has no step)
                const bool none = L == 0.f;
                const int slot = 2 * blockIdx.x + (p.k0 == 0 ? 1 : 0);
                const int row = sub * tok * G + r;
                const uint32_t oc = tmem + lanes + T::kO + (pl.two ? w * HD : 0);
                const int from = join ? w * (HD / 2) : 0, to = join ? from + HD / 2 : HD;
                uint8_t *stage = outs + warp * T::kOutBytes;
#pragma unroll 1
                for (int j = from; j < to; j += 32) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(oc + j, v);
                    tmem_ld_wait();
                    float y[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = none ? 0.f : __uint_as_float(v[e]) * f0;
                    if (both) {
                        tmem_ld_32x32b_x32(oc + HD + j, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (f1 != 0.f) y[e] = fmaf(__uint_as_float(v[e]), f1, y[e]);
                    }
                    if (!whole) {
                        // [dim / 4][row][4]: neighbouring threads write neighbouring 16 bytes
                        float *pp = a.part_o + (int64_t)slot * T::kRows * HD + row * 4;
                        if (r < valid) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                *reinterpret_cast<float4 *>(pp + ((j + e) >> 2) * (T::kRows * 4)) =
                                    make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                        }
                        continue;
                    }
                    // a warp's 32 rows x 32 dims turn in shared memory into stores of 64
                    // bytes of a row (16-byte chunks swizzled by the row)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<uint4 *>(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) =
                            make_uint4(pack_t2<F16>(y[8 * e], y[8 * e + 1]),
                                       pack_t2<F16>(y[8 * e + 2], y[8 * e + 3]),
                                       pack_t2<F16>(y[8 * e + 4], y[8 * e + 5]),
                                       pack_t2<F16>(y[8 * e + 6], y[8 * e + 7]));
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), e = lane & 3;
                        const int R = (warp & 3) * 32 + rr;
                        const int t = (int)((uint32_t)R * inv_g >> 16);
                        if (R < valid)
                            *reinterpret_cast<uint4 *>(
                                a.out + (int64_t)(p.s.q0 + t0 + t) * a.out_ld +
                                (int64_t)(p.h * G + R - t * G) * HD + j + e * 8) =
                                *reinterpret_cast<const uint4 *>(
                                    stage + rr * 64 + ((e ^ ((rr >> 1) & 3)) << 4));
                    }
                }
                if (!whole && r < valid && (!join || w == 0))
                    *reinterpret_cast<float2 *>(a.part_ml + ((int64_t)slot * T::kRows + row) * 2) =
                        make_float2(M * cs, L);
            }
            if (threadIdx.x == 0 && ok && job.p.parts > 0)
                a.notes[blockIdx.x] = SplitNote{p.s.q0 + p.t0, p.h * G, p.t1 - p.t0, p.parts};
            // (the next piece's first product into O waits for this warpgroup's weights,
            // and the barrier above for both warpgroups)
            tc_fence_before();
            blocks += pl.n;
            pvs += steps;
            __syncwarp();
            if (lane == 0) mbar_arrive(&job_empty[pieces & 1]);
            ++pieces;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort) {  // given up: the copies in flight end before this CTA does (they take microseconds)
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 10000000ull) {
        }
    }
    if (warp == T::kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int HD, bool F16>
cudaError_t run_tiles(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                      cudaStream_t st) {
    const int G = a.n_heads / a.n_kv;
    CUtensorMap mq;
    if (!make_map_rows(&mq, F16, a.q, HD, a.n_heads, a.pb.n_tokens, a.q_ld, G, kBlock / G))
        return cudaErrorInvalidValue;
    auto kern = paged_tiles_kernel<HD, F16>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, Tc<HD>::kSmem, allowed);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3((unsigned)sm_count()), Tc<HD>::kThreads, Tc<HD>::kSmem, st, mq, mk,
                      mv, a);
}

}  // namespace

int paged_tiles_rows(int head_dim) { return head_dim == 256 ? Tc<256>::kRows : Tc<128>::kRows; }

cudaError_t launch_paged_tiles(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                               int hd, bool f16, cudaStream_t st) {
    if (f16) {
        if (hd == 64) return run_tiles<64, true>(a, mk, mv, st);
        if (hd == 128) return run_tiles<128, true>(a, mk, mv, st);
        return run_tiles<256, true>(a, mk, mv, st);
    }
    if (hd == 64) return run_tiles<64, false>(a, mk, mv, st);
    if (hd == 128) return run_tiles<128, false>(a, mk, mv, st);
    return run_tiles<256, false>(a, mk, mv, st);
}

}  // namespace nq
