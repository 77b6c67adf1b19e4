// attn_shared.cu -- attention of many sequences over one shared prefix and a
// suffix of each one's own, on B200 (sm_100a).
//
// For sequence i, query head h (kv head h / G, G = n_head / n_kv) and its keys
// t = the prefix rows 0 .. P-1, then rows 0 .. len_i - 1 of its cache slot:
//   out[i][h] = sum_t p_t V_t / sum_t p_t,   p_t = exp(scale q . K_t - max)
// (the attention of Tsuskov/talos src/model/llama.rs:135-155 per sequence). No
// key at all gives zeros.
//
// The queries of all sequences that share a kv head are the rows of one matrix:
// 128 / G sequences fill a row tile of 128 rows, and the prefix's keys are read
// once per row tile instead of once per sequence and head. The sequences'
// suffixes follow the prefix in the row tile's list of key tiles (KT keys; a
// suffix starts a tile of its own, so one sequence's infinities or NaN never meet
// another's rows); a row takes part in the prefix's tiles and its own. So prefix
// and suffix are the same work, and each CTA takes an equal run of a row tile's
// list over the kv heads; a run that does not hold a whole (row tile, kv head)
// leaves (max, sum, O) partials that k_attn_merge adds in order.
//
// Per tile: S = Q K^T and O = P V on the 5th-generation tensor cores
// (tcgen05.mma kind::f16, M 128), S and O in tensor memory, P written back over S
// in 16 bits as the A operand. The softmax keeps a running maximum m, rounded up
// to an integer (base 2), so every rescaling is by an exact power of two; O is
// added up in registers in f32 (the tensor core only sums one tile: its
// accumulation truncates).
//
// Precision. f16 / bf16 queries: one product each, P rounded to 16 bits (half a
// step of 2^-11 / 2^-8 relative per weight, averaged by the sum; the row sum uses
// the unrounded weights), f32 everywhere else. f32 queries: q is scaled by a power
// of two into [2^14, 2^15) at its largest element and split into f16 hi + lo (22
// bits), and so is P; an f32 cache's rows too, with a power of two per key that
// multiplies its score (K) or moves its weight's exponent (V), so no input
// overflows f16 and small ones keep their bits. lo x lo (2^-22) is left out.
//
// Roles of the 16 warps (one CTA per SM):
//  * warps 0-7: softmax. Warps w and w + 4 share the rows 32 w .. 32 w + 31 (their
//    TMEM lanes), one half of the tile's keys and of the head's dims each; they
//    exchange row maxima in shared memory.
//  * warps 8-14: producers. 16-byte cp.async copies of K / V rows, zero-filled
//    behind the last key, straight into the swizzled operand tiles (16-bit caches)
//    or into a per-warp ring whose rows the same lanes then scale and split (f32).
//  * warp 15: TMEM allocation; one lane issues the MMAs: QK of tile j ahead of PV
//    of tile j - 1, so that the softmax of one tile runs beside the products of its
//    neighbours.
// Bound: HBM (the keys once) up to one row tile; above, softmax issue slots.
//
// Every wait is bounded (2 s); on expiry a CTA flag makes all roles run on without
// waiting or multiplying, and the rows come out as NaN.
#include <math.h>

#include "ops.cuh"
#include "ptx.cuh"

namespace talos {

constexpr int AS_THREADS = 512;
constexpr int AS_NP = 7;       // producer warps
constexpr int AS_PW0 = 8, AS_MMA = 15;
constexpr int AS_ROWS = 128;   // rows per tile = TMEM lanes
constexpr int AS_SOFT_REGS = 184, AS_REST_REGS = 72;  // 256 x (184 + 72) = 512 x 128
constexpr int AS_MISC = 12 * 1024;
constexpr int AS_SMEM = 227 * 1024;
constexpr float AS_LOG2E = 1.4426950408889634f;

// MODE: types of (q, cache): 0 (f32, f32), 1 (f32, f16), 2 (f16, f16), 3 (bf16, bf16)
template <int MODE, int DP>
struct AsCfg {
    static constexpr bool QF32 = MODE <= 1, KF32 = MODE == 0, BF = MODE == 3;
    static constexpr int NQ = QF32 ? 2 : 1;  // planes (hi, lo) of Q and P
    static constexpr int NK = KF32 ? 2 : 1;  // of K and V
    static constexpr int KT = KF32 ? 64 : 128;  // keys per tile
    static constexpr int ES = KF32 ? 4 : 2;     // bytes of a cache element
    static constexpr int QPLANE = AS_ROWS * DP * 2, KPLANE = KT * DP * 2;
    static constexpr int CPR = DP * ES / 16;   // 16-byte chunks of a cache row
    static constexpr int RPW = 32 / CPR;       // rows per warp copy
    static constexpr int ITERS = (KT / RPW + AS_NP - 1) / AS_NP;  // copies per warp and tile
    static constexpr int RAWD = 24;            // f32: rows in flight per warp
    static constexpr int RAW = KF32 ? AS_NP * RAWD * 512 : 0;
    static constexpr int FIT = (AS_SMEM - AS_MISC - NQ * QPLANE - RAW) / (2 * NK * KPLANE);
    static constexpr int NS = KF32 ? 1 : (FIT > 4 ? 4 : FIT);  // K / V stages
    static constexpr int SMEM = NQ * QPLANE + NS * 2 * NK * KPLANE + RAW + AS_MISC;
    static constexpr int S_COLS = KT;          // TMEM columns of one S buffer; P lies over it
    static constexpr int O_COL = 2 * KT;       // first column of the two O buffers
    static_assert(NS >= 1 && SMEM <= AS_SMEM, "shared memory");
    static_assert(2 * KT + 2 * DP <= 512, "tensor memory");
    static_assert(RPW * ITERS <= 32, "one lane per row of a warp");
};

struct AsMisc {
    uint64_t q_full, q_empty, k_full[4], k_empty[4], v_full[4], v_empty[4];
    uint64_t s_full[2], p_full[2], o_full[2], o_empty[2], done;
    uint32_t tmem;
    int fail;
    int rt, b0, nb, tpg;     // row tile of this CTA, its first CTA and CTA count, tiles per kv head
    int ntile_p, total;      // prefix tiles; tiles of the row tile
    int cum[AS_ROWS + 1];    // suffix tiles before each of the row tile's sequences
    int len[AS_ROWS], slot[AS_ROWS];
    float qsc[2][AS_ROWS];   // row scale: scale * log2(e) * 2^(exponent of q)
    float mx[2][2][AS_ROWS], mx2[2][2][AS_ROWS];  // [tile parity][half] row maxima
    float lx[2][AS_ROWS];
    alignas(16) float ksc[4][64];   // f32 cache: 2^(key's exponent)
    alignas(16) float2 vsc[4][64];  // f32 cache: value row's exponent e and 2^e
    int scan[16];
};
static_assert(sizeof(AsMisc) <= AS_MISC, "misc area");

// ---------------------------------------------------------------- PTX

__device__ __forceinline__ void as_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void as_tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void as_tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void as_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// 128-byte-swizzled operand tiles: 128-byte rows, chunk c of row r at c ^ (r % 8),
// 8-row atoms 1024 bytes apart (SBO). K-major (Q, K): LBO unused. MN-major (V: the
// 128-byte rows are keys, the K dimension): LBO = bytes between blocks of 64 dims.
__device__ __forceinline__ uint64_t as_desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// f32 accumulators, f16 or bf16 operands, M 128, B K-major or MN-major.
__host__ __device__ constexpr uint32_t as_idesc(int n, bool bf, bool b_mn) {
    return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(AS_ROWS >> 4) << 24);
}
__device__ __forceinline__ void as_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void as_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void as_ld32(uint32_t t, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void as_st8(uint32_t t, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void as_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void as_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void as_pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void as_cp16(uint32_t dst, const void* src, uint32_t bytes) {  // the rest of 16: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void as_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void as_cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float as_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF>
__device__ __forceinline__ uint32_t as_pack(float a, float b) {
    if constexpr (BF) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ void as_split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = as_pack<false>(a - f.x, b - f.y);
}
// The exponent e of the largest |x| (its bits), as used for scaling: x 2^(14 - e)
// lies in [2^14, 2^15); kept where 2^(14 - e) and 2^(e - 14) are normal.
__device__ __forceinline__ int as_exponent(uint32_t abs_bits) {
    const int e = (int)(abs_bits >> 23) - 127;
    return e < -112 ? -112 : e;
}
__device__ __forceinline__ float as_pow2(int e) { return __int_as_float((e + 127) << 23); }

// Bounded wait; once the CTA has failed, no wait waits.
__device__ __forceinline__ void as_wait(AsMisc* m, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(bar, parity)) return;
        if (*(volatile int*)&m->fail) return;
        if (globaltimer_ns() - t0 > 2000000000ull) {
            *(volatile int*)&m->fail = 1;
            return;
        }
    }
}

// First row of part i of n rows cut into nb even parts.
__device__ __forceinline__ int as_part(int i, int n, int nb) { return (int)((long long)i * n / nb); }

__device__ __forceinline__ int as_len(const AttnSharedArgs& a, int seq, int prefix) {
    int len;
    if (a.pos) len = (int)a.pos[seq] + 1 - prefix;  // batched step: positions count the prefix
    else len = a.lens[seq];
    return len < 0 ? 0 : (len > a.slot_len ? a.slot_len : len);
}
__device__ __forceinline__ int as_slot(const AttnSharedArgs& a, int seq) {
    const int s = a.slots ? a.slots[seq] : seq;
    return s >= 0 && s < a.n_slots ? s : -1;
}

// The sequence (within its row tile) that suffix tile t belongs to: the last one
// that starts at or before it and has any (empty suffixes start where the next does).
__device__ __forceinline__ int as_owner(const AsMisc* m, int nseq, int t) {
    int lo = 0, hi = nseq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (m->cum[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Suffix tiles of sequences seq0 .. seq0 + ns - 1, summed by a warp.
__device__ __forceinline__ int as_suffix_tiles(const AttnSharedArgs& a, int seq0, int ns, int prefix, int KT) {
    int t = 0;
    for (int i = threadIdx.x & 31; i < ns; i += 32)
        if (as_slot(a, seq0 + i) >= 0) t += (as_len(a, seq0 + i, prefix) + KT - 1) / KT;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// ---------------------------------------------------------------- the kernel

template <int MODE, int DP>
__global__ void __launch_bounds__(AS_THREADS, 1) k_attn_shared(const __grid_constant__ AttnSharedArgs a) {
    using C = AsCfg<MODE, DP>;
    constexpr int KT = C::KT;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + C::NQ * C::QPLANE;            // [NS][planes]
    uint8_t* sV = sK + C::NS * C::NK * C::KPLANE;    // [NS][planes]
    uint8_t* sR = sV + C::NS * C::NK * C::KPLANE;    // f32: raw rows [producer warp][RAWD][512]
    AsMisc* m = (AsMisc*)(sR + C::RAW);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    const int n = a.n_dev ? *a.n_dev : a.n;
    const int prefix = a.prefix_dev ? (int)*a.prefix_dev : a.prefix;
    const int G = a.group, spt = AS_ROWS / G;          // sequences per row tile
    const int R = (n + spt - 1) / spt;
    const int ntp = (prefix + KT - 1) / KT;

    // ---- this CTA's row tile and run of tiles
    if (tid == 0) m->fail = 0;
    if (R > 1 && !a.whole) {
        // CTAs in proportion to the row tiles' work: row tile r has CTAs b(r) ..
        // b(r + 1) - 1, b(r) = r + (N - R) * (tiles before r) / (all tiles)
        const int N = gridDim.x;
        long long total = 0, before = 0;
        int found = -1, b_lo = 0, b_hi = 0;
        for (int pass = 0; pass < 2; ++pass) {
            before = 0;
            for (int r0 = 0; r0 < R; r0 += 16) {
                const int r = r0 + warp;  // a warp sums one row tile's suffix tiles
                const int own = as_suffix_tiles(a, r * spt, min(spt, n - r * spt), prefix, KT);
                __syncthreads();
                if (lane == 0) m->scan[warp] = r < R ? (ntp + own) * a.n_kv : 0;
                __syncthreads();
                for (int k = 0; k < 16 && r0 + k < R; ++k) {
                    const int t = m->scan[k];
                    if (pass == 1) {
                        const int lo = r0 + k + (int)(total ? (long long)(N - R) * before / total : 0);
                        const int hi = r0 + k + 1 + (int)(total ? (long long)(N - R) * (before + t) / total : 0);
                        if (blockIdx.x == 0 && tid == 0) a.plan[2 * (r0 + k)] = lo, a.plan[2 * (r0 + k) + 1] = hi - lo;
                        if ((int)blockIdx.x >= lo && (int)blockIdx.x < hi) found = r0 + k, b_lo = lo, b_hi = hi;
                    }
                    before += t;
                }
            }
            total = before;
        }
        if (tid == 0) m->rt = found, m->b0 = b_lo, m->nb = b_hi - b_lo;
    } else if (tid == 0) {
        // one row tile: all CTAs; or (whole) one CTA per (row tile, kv head)
        m->rt = a.whole ? (int)blockIdx.x / a.n_kv : 0;
        m->b0 = a.whole ? m->rt * a.n_kv : 0;
        m->nb = a.whole ? a.n_kv : (int)gridDim.x;
        if (!a.whole && blockIdx.x == 0) a.plan[0] = 0, a.plan[1] = (int)gridDim.x;
    }
    __syncthreads();
    const int rt = m->rt, b0 = m->b0, nb = m->nb;
    if (rt < 0 || rt >= R) return;
    const int seq0 = rt * spt, nseq = min(spt, n - seq0);
    if (warp == 0) {  // the row tile's suffix list
        int run = 0;
        for (int i0 = 0; i0 < nseq; i0 += 32) {
            const int i = i0 + lane;
            int slot = -1, len = 0;
            if (i < nseq) {
                slot = as_slot(a, seq0 + i);
                len = slot >= 0 ? as_len(a, seq0 + i, prefix) : 0;
            }
            const int nt = (len + KT - 1) / KT;
            int x = nt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (i < nseq) m->cum[i] = run + x - nt, m->len[i] = len, m->slot[i] = slot;
            run += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) {
            m->cum[nseq] = run;
            m->tpg = ntp + run;
        }
    }
    if (tid == 32) {
        mbar_init(&m->q_full, AS_NP);
        mbar_init(&m->q_empty, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&m->k_full[i], AS_NP);
            mbar_init(&m->k_empty[i], 1);
            mbar_init(&m->v_full[i], AS_NP);
            mbar_init(&m->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&m->s_full[i], 1);
            mbar_init(&m->p_full[i], 8);
            mbar_init(&m->o_full[i], 1);
            mbar_init(&m->o_empty[i], 8);
        }
        mbar_init(&m->done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int tpg = m->tpg, total = tpg * a.n_kv;  // tiles per kv head, tiles of the row tile
    const int rank = (int)blockIdx.x - b0;
    const int t0 = as_part(rank, total, nb), t1 = as_part(rank + 1, total, nb);
    if (tpg == 0) {
        // no key in the whole row tile: zeros
        if (rank == 0)
            for (int i = tid; i < nseq * G * a.n_kv * a.hd; i += AS_THREADS) {
                const int d = i % a.hd, h = i / a.hd % (G * a.n_kv), s = seq0 + i / a.hd / (G * a.n_kv);
                const size_t at = (size_t)s * a.out_sn + (size_t)h * a.out_sh + d;
                if (C::QF32) ((float*)a.out)[at] = 0.f;
                else ((uint16_t*)a.out)[at] = 0;
            }
        return;
    }
    if (t0 >= t1) return;
    if (warp == AS_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&m->tmem)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    as_tc_before();
    __syncthreads();
    as_tc_after();
    const uint32_t tmem = m->tmem;
    const int rows = nseq * G;  // live rows

    if (warp >= AS_PW0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AS_REST_REGS));
        if (warp == AS_MMA) {
            // ------------------------------------------------ MMA issuer
            if (lane == 0) {
                const int ksteps = (a.hd + 15) / 16;
                const uint32_t id_qk = as_idesc(KT, C::BF, false), id_pv = as_idesc(ksteps * 16, C::BF, true);
                const uint32_t q_hi = smem_u32(sQ), q_lo = q_hi + C::QPLANE;
                int j = 0, seg = -1, cur = -1;
                auto issue_pv = [&](int i) {  // tile i (counted from the CTA's first)
                    const int sv = i % C::NS, bf = i & 1;
                    as_wait(m, &m->p_full[bf], (i >> 1) & 1);
                    as_wait(m, &m->v_full[sv], (i / C::NS) & 1);
                    as_wait(m, &m->o_empty[bf], ((i >> 1) & 1) ^ 1);
                    as_tc_after();
                    if (!*(volatile int*)&m->fail) {
                        const uint32_t d = tmem + C::O_COL + bf * DP, p = tmem + bf * C::S_COLS;
                        const uint32_t v = smem_u32(sV + sv * C::NK * C::KPLANE);
                        uint32_t acc = 0;
                        // the small terms first
#pragma unroll
                        for (int pr = C::NQ + C::NK - 2; pr >= 0; --pr) {
                            const bool p_lo = C::NQ == 2 && pr == 1, v_lo = pr == 2;
                            const uint32_t pa = p + (p_lo ? KT / 2 : 0);
                            const uint64_t vd = as_desc(v + (v_lo ? C::KPLANE : 0), KT * 128);
#pragma unroll
                            for (int ks = 0; ks < KT / 16; ++ks) {
                                as_mma_ts(d, pa + 8 * ks, vd + (uint64_t)(ks * 2048 >> 4), id_pv, acc);
                                acc = 1;
                            }
                        }
                    }
                    as_commit(&m->v_empty[sv]);
                    as_commit(&m->o_full[bf]);
                };
                for (int t = t0; t < t1; ++t, ++j) {
                    const int kvh = t / tpg;
                    if (kvh != cur) {
                        cur = kvh, ++seg;
                        as_wait(m, &m->q_full, seg & 1);
                    }
                    const int sk = j % C::NS, bf = j & 1;
                    as_wait(m, &m->k_full[sk], (j / C::NS) & 1);
                    if (j >= 2) as_wait(m, &m->o_full[bf], ((j - 2) >> 1) & 1);  // P over this S buffer was read
                    as_tc_after();
                    if (!*(volatile int*)&m->fail) {
                        const uint32_t d = tmem + bf * C::S_COLS;
                        const uint32_t k = smem_u32(sK + sk * C::NK * C::KPLANE);
                        uint32_t acc = 0;
#pragma unroll
                        for (int pr = C::NQ + C::NK - 2; pr >= 0; --pr) {
                            const bool ql = C::NQ == 2 && pr == 1, kl = pr == 2;
                            const uint32_t qa = ql ? q_lo : q_hi, ka = k + (kl ? C::KPLANE : 0);
                            for (int ks = 0; ks < ksteps; ++ks) {
                                const uint64_t qd = as_desc(qa + (ks >> 2) * (AS_ROWS * 128) + (ks & 3) * 32, 16);
                                const uint64_t kd = as_desc(ka + (ks >> 2) * (KT * 128) + (ks & 3) * 32, 16);
                                as_mma_ss(d, qd, kd, id_qk, acc);
                                acc = 1;
                            }
                        }
                    }
                    as_commit(&m->k_empty[sk]);
                    as_commit(&m->s_full[bf]);
                    if (t + 1 == t1 || (t + 1) / tpg != kvh) as_commit(&m->q_empty);  // the queries may be replaced
                    if (j > 0) issue_pv(j - 1);
                }
                issue_pv(j - 1);
                as_commit(&m->done);
                as_wait(m, &m->done, 0);  // nothing in flight when TMEM is freed
            }
            __syncwarp();
        } else {
            // ------------------------------------------------ producers
            const int w = warp - AS_PW0;
            const int chunk = lane % C::CPR, sub = lane / C::CPR;
            const uint32_t row_bytes = (uint32_t)a.hd * C::ES;
            const uint32_t live_bytes = (uint32_t)chunk * 16 < row_bytes ? 16u : 0u;
            // the lane's row of a tile: its address, or none
            struct Rows {
                const uint8_t *k, *v;
                bool ok;
            };
            auto row_of = [&](int t) {
                Rows r{(const uint8_t*)a.q, (const uint8_t*)a.q, false};
                const int kvh = t / tpg, off = t % tpg;
                const int row = (w + AS_NP * (lane / C::RPW)) * C::RPW + lane % C::RPW;
                if (lane >= C::RPW * C::ITERS || row >= KT) return r;
                if (off < ntp) {
                    const int key = off * KT + row;
                    if (key < prefix) {
                        const size_t at = ((size_t)key * a.pre_st + (size_t)kvh * a.pre_sh) * C::ES;
                        r = Rows{(const uint8_t*)a.kp + at, (const uint8_t*)a.vp + at, true};
                    }
                } else {
                    const int i = as_owner(m, nseq, off - ntp), key = (off - ntp - m->cum[i]) * KT + row;
                    if (key < m->len[i]) {
                        const size_t at = ((size_t)m->slot[i] * a.slot_ss +
                                           (size_t)(key + a.slot_row0 * prefix) * a.slot_st +
                                           (size_t)kvh * a.slot_sh) * C::ES;
                        r = Rows{(const uint8_t*)a.k + at, (const uint8_t*)a.v + at, true};
                    }
                }
                return r;
            };
            // the queries of kv head kvh into sQ
            auto load_q = [&](int kvh, int seg) {
                if (seg > 0) as_wait(m, &m->q_empty, (seg - 1) & 1);
                if constexpr (C::QF32) {
                    constexpr int QC = DP / 4, QR = 32 / QC;  // float4 chunks of a row, rows per warp
                    constexpr int QI = (AS_ROWS / QR + AS_NP - 1) / AS_NP, QB = 5;
                    const int ch = lane % QC;
                    for (int i0 = 0; i0 < QI; i0 += QB) {
                        float4 v[QB];
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const int r = (w + AS_NP * (i0 + i)) * QR + lane / QC;
                            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (r < rows && 4 * ch < a.hd)
                                v[i] = *(const float4*)((const float*)a.q + (size_t)(seq0 + r / G) * a.q_sn +
                                                        (size_t)(kvh * G + r % G) * a.q_sh + 4 * ch);
                        }
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const int r = (w + AS_NP * (i0 + i)) * QR + lane / QC;
                            uint32_t b = __float_as_uint(fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)),
                                                               fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
#pragma unroll
                            for (int o = QC / 2; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
                            if (r >= rows) continue;
                            const int e = as_exponent(b);
                            const float f = as_pow2(14 - e);
                            uint2 hi, lo;
                            as_split(v[i].x * f, v[i].y * f, hi.x, lo.x);
                            as_split(v[i].z * f, v[i].w * f, hi.y, lo.y);
                            uint8_t* dst = sQ + (ch / 16) * (AS_ROWS * 128) + r * 128 +
                                           (((ch % 16 / 2) ^ (r & 7)) << 4) + (ch & 1) * 8;
                            *(uint2*)dst = hi;
                            *(uint2*)(dst + C::QPLANE) = lo;
                            if (ch == 0) m->qsc[seg & 1][r] = as_pow2(e - 14) * (a.scale * AS_LOG2E);
                        }
                    }
                } else {
                    constexpr int QC = DP / 8, QR = 32 / QC;
                    constexpr int QI = (AS_ROWS / QR + AS_NP - 1) / AS_NP, QB = 5;
                    const int ch = lane % QC;
                    for (int i0 = 0; i0 < QI; i0 += QB) {
                        uint4 v[QB];
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const int r = (w + AS_NP * (i0 + i)) * QR + lane / QC;
                            v[i] = make_uint4(0, 0, 0, 0);
                            if (r < rows && 8 * ch < a.hd)
                                v[i] = *(const uint4*)((const uint16_t*)a.q + (size_t)(seq0 + r / G) * a.q_sn +
                                                       (size_t)(kvh * G + r % G) * a.q_sh + 8 * ch);
                        }
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const int r = (w + AS_NP * (i0 + i)) * QR + lane / QC;
                            if (r < rows)
                                *(uint4*)(sQ + (ch / 8) * (AS_ROWS * 128) + r * 128 + (((ch % 8) ^ (r & 7)) << 4)) = v[i];
                        }
                    }
                }
                as_fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&m->q_full);
            };

            if constexpr (!C::KF32) {
                // jobs: K then V of each tile; up to LAG jobs stay in flight. PV of a tile is
                // issued behind QK of the next one, so a V stage is free again only after the
                // K job 2 NS - 1 before has landed: LAG is at most 2 NS - 2
                constexpr int LAG = 2 * C::NS - 2;
                static_assert(LAG >= 1, "two stages at least");
                int issued = 0, landed = 0;  // jobs
                auto land = [&]() {  // the oldest job in flight has arrived
                    as_fence_async();
                    __syncwarp();
                    const int i = landed >> 1;
                    if (lane == 0) mbar_arrive(landed & 1 ? &m->v_full[i % C::NS] : &m->k_full[i % C::NS]);
                    ++landed;
                };
                auto issue = [&](const Rows& r, bool is_v) {
                    const int i = issued >> 1, s = i % C::NS;
                    as_wait(m, is_v ? &m->v_empty[s] : &m->k_empty[s], ((i / C::NS) & 1) ^ 1);
                    const uint32_t dst = smem_u32((is_v ? sV : sK) + s * C::KPLANE) + (chunk / 8) * (KT * 128);
                    const unsigned long long p = (unsigned long long)(is_v ? r.v : r.k);
#pragma unroll
                    for (int it = 0; it < C::ITERS; ++it) {
                        const int from = it * C::RPW + sub;
                        const uint8_t* src = (const uint8_t*)__shfl_sync(0xffffffffu, p, from);
                        const bool ok = __shfl_sync(0xffffffffu, (int)r.ok, from);
                        const int row = (w + AS_NP * it) * C::RPW + sub;
                        if (row < KT) {
                            const uint32_t nb_ = ok ? live_bytes : 0u;
                            as_cp16(dst + row * 128 + (((chunk % 8) ^ (row & 7)) << 4), nb_ ? src + chunk * 16 : a.q, nb_);
                        }
                    }
                    as_cp_commit();
                    ++issued;
                };
                int cur = -1, seg = -1;
                for (int t = t0; t < t1; ++t) {
                    const bool fresh = t / tpg != cur;
                    if (fresh && seg >= 0) {  // the queries wait for every product of the segment before
                        as_cp_wait<0>();
                        while (landed < issued) land();
                    }
                    const Rows r = row_of(t);
                    issue(r, false);
                    if (issued - landed > LAG) {
                        as_cp_wait<LAG>();
                        land();
                    }
                    issue(r, true);
                    if (fresh) cur = t / tpg, load_q(cur, ++seg);
                    if (issued - landed > LAG) {
                        as_cp_wait<LAG>();
                        land();
                    }
                }
                as_cp_wait<0>();
                while (landed < issued) land();
            } else {
                // f32 rows: a lane's 16 bytes go through its own ring slots, RAWD - 1
                // copies ahead of the conversion; K rows of a tile, then its V rows
                const uint32_t ring = smem_u32(sR) + w * C::RAWD * 512 + lane * 16;
                const int total_it = (t1 - t0) * 2 * C::ITERS;
                int it_i = 0, t_i = t0, half_i = 0;  // issue cursor
                uint32_t slot_i = 0, slot_c = 0;
                Rows r_i = row_of(t0);
                auto issue = [&]() {
                    if (t_i < t1) {
                        const unsigned long long p = (unsigned long long)(half_i ? r_i.v : r_i.k);
                        const int from = it_i * C::RPW + sub;
                        const uint8_t* src = (const uint8_t*)__shfl_sync(0xffffffffu, p, from);
                        const bool ok = __shfl_sync(0xffffffffu, (int)r_i.ok, from);
                        const uint32_t nb_ = ok ? live_bytes : 0u;
                        as_cp16(ring + slot_i * 512, nb_ ? src + chunk * 16 : a.q, nb_);
                        slot_i = slot_i + 1 == C::RAWD ? 0 : slot_i + 1;
                        if (++it_i == C::ITERS) {
                            it_i = 0;
                            if (half_i) {
                                if (++t_i < t1) r_i = row_of(t_i);
                            }
                            half_i ^= 1;
                        }
                    }
                    as_cp_commit();  // (empty at the end: the count of groups stays in step)
                };
                for (int i = 0; i < C::RAWD - 1; ++i) issue();
                int cur = -1, seg = -1, it_c = 0, half_c = 0, t_c = t0, j = 0;
                for (int c = 0; c < total_it; ++c) {
                    issue();
                    if (it_c == 0) {
                        if (half_c == 0 && t_c / tpg != cur) cur = t_c / tpg, load_q(cur, ++seg);
                        if (j > 0) as_wait(m, half_c ? &m->v_empty[0] : &m->k_empty[0], (j - 1) & 1);
                    }
                    as_cp_wait<C::RAWD - 1>();
                    float4 v;
                    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                                 : "r"(ring + slot_c * 512)
                                 : "memory");
                    slot_c = slot_c + 1 == C::RAWD ? 0 : slot_c + 1;
                    const int row = (w + AS_NP * it_c) * C::RPW + sub;
                    uint32_t b = __float_as_uint(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                    if constexpr (C::RPW == 1) {
                        b = __reduce_max_sync(0xffffffffu, b);
                    } else {
#pragma unroll
                        for (int o = C::CPR / 2; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
                    }
                    if (row < KT) {
                        const int e = as_exponent(b);
                        const float f = as_pow2(14 - e);
                        uint2 hi, lo;
                        as_split(v.x * f, v.y * f, hi.x, lo.x);
                        as_split(v.z * f, v.w * f, hi.y, lo.y);
                        uint8_t* dst = (half_c ? sV : sK) + (chunk / 16) * (KT * 128) + row * 128 +
                                       (((chunk % 16 / 2) ^ (row & 7)) << 4) + (chunk & 1) * 8;
                        *(uint2*)dst = hi;
                        *(uint2*)(dst + C::KPLANE) = lo;
                        if (chunk == 0) {
                            if (half_c) m->vsc[j & 3][row] = make_float2((float)(e - 14), as_pow2(e - 14));
                            else m->ksc[j & 3][row] = as_pow2(e - 14);
                        }
                    }
                    if (++it_c == C::ITERS) {
                        as_fence_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(half_c ? &m->v_full[0] : &m->k_full[0]);
                        it_c = 0;
                        if (half_c) ++t_c, ++j;
                        half_c ^= 1;
                    }
                }
                as_cp_wait<0>();
            }
        }
    } else {
        // ------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AS_SOFT_REGS));
        const int half = warp >> 2, q4 = warp & 3;
        const int row = q4 * 32 + lane, sq = row / G;
        const bool live = row < rows;
        const uint32_t lane_base = tmem + ((uint32_t)(q4 * 32) << 16);
        constexpr int HC = KT / 2, HD = DP / 2;  // this thread's keys of a tile, dims of the output
        constexpr float OFF = C::BF ? 0.f : 14.f;  // f16 weights: 2^14 at the maximum keeps small ones normal
        float o[HD];
        float mrun = -INFINITY, Mrun = -INFINITY, lsum = 0.f, cprev = 1.f, qs = 0.f;
        bool prev_act = false, prev_any = false;
        const int own0 = live ? m->cum[sq] : 0, own = live ? m->len[sq] : 0;  // its first suffix tile, its keys

        auto add_o = [&](int i) {  // o = o * cprev + O of tile i
            as_wait(m, &m->o_full[i & 1], (i >> 1) & 1);
            as_tc_after();
            if (prev_any) {
                const uint32_t src = lane_base + C::O_COL + (i & 1) * DP + half * HD;
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    float x[32];
                    as_ld32(src + c, x);
                    as_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[c + k] = prev_act ? fmaf(o[c + k], cprev, x[k]) : o[c + k];
                }
            }
            as_tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&m->o_empty[i & 1]);
        };

        int j = 0, cur = -1, seg = -1, seg_t0 = t0;
        for (int t = t0; t < t1; ++t, ++j) {
            const int kvh = t / tpg, off = t % tpg, bf = j & 1;
            const bool first = kvh != cur;
            if (first) {
                cur = kvh, ++seg, seg_t0 = t;
#pragma unroll
                for (int k = 0; k < HD; ++k) o[k] = 0.f;
                mrun = Mrun = -INFINITY;
                lsum = 0.f;
            }
            // the row's keys of this tile: the first hi
            int hi = 0;
            if (off < ntp) {
                if (live) hi = min(KT, prefix - off * KT);
            } else if (off - ntp >= own0) {
                hi = (int)min((long long)KT, own - (long long)(off - ntp - own0) * KT);
            }
            const bool act = hi > 0;
            const bool any = __any_sync(0xffffffffu, act);
            as_wait(m, &m->s_full[bf], (j >> 1) & 1);
            if (C::KF32) as_wait(m, &m->v_full[0], j & 1);  // the values' exponents
            as_tc_after();
            if (first) qs = C::QF32 ? (live ? m->qsc[seg & 1][row] : 0.f) : a.scale * AS_LOG2E;
            float cnew = 1.f;
            if (any) {
                float s[HC];
                const uint32_t sb = lane_base + bf * C::S_COLS;
#pragma unroll
                for (int c = 0; c < HC; c += 32) as_ld32(sb + half * HC + c, s + c);
                as_wait_ld();
                const int h0 = hi - half * HC;
                const bool full = __all_sync(0xffffffffu, h0 >= HC);
                float mt = -INFINITY, Mt = -INFINITY;
                if (C::KF32) {
#pragma unroll
                    for (int k = 0; k < HC; k += 4) {
                        const float4 ks = *(const float4*)&m->ksc[j & 3][half * HC + k];
                        s[k] *= ks.x, s[k + 1] *= ks.y, s[k + 2] *= ks.z, s[k + 3] *= ks.w;
                    }
                }
                // (s stays unscaled; the scaled maximum is the maximum of the scaled, qs > 0)
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < HC; ++k) m4[k & 3] = fmaxf(m4[k & 3], full || k < h0 ? s[k] : -INFINITY);
                mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * qs;
                if (C::KF32) {
#pragma unroll
                    for (int k = 0; k < HC; k += 2) {
                        const float4 vs = *(const float4*)&m->vsc[j & 3][half * HC + k];
                        Mt = fmaxf(Mt, fmaxf(full || k < h0 ? fmaf(s[k], qs, vs.x) : -INFINITY,
                                             full || k + 1 < h0 ? fmaf(s[k + 1], qs, vs.z) : -INFINITY));
                    }
                }
                m->mx[bf][half][row] = mt;
                if (C::KF32) m->mx2[bf][half][row] = Mt;
                as_pair_sync(1 + q4);  // (also: both halves of S are read, P may overwrite them)
                mt = fmaxf(mt, m->mx[bf][half ^ 1][row]);
                const float mnew = fmaxf(mrun, ceilf(mt));
                float fv = 0.f, Mnew = Mrun;
                if (C::KF32) {
                    Mt = fmaxf(Mt, m->mx2[bf][half ^ 1][row]);
                    Mnew = fmaxf(Mrun, ceilf(Mt));
                }
                if (act) {
                    // integer exponents: exact powers of two (0 on the first tile)
                    const float cl = as_ex2(mrun - mnew);
                    cnew = C::KF32 ? as_ex2(Mrun - Mnew) : cl;
                    lsum *= cl;
                    mrun = mnew, Mrun = Mnew;
                    if (C::KF32) fv = mnew - Mnew + OFF;
                }
                const float sub = C::KF32 ? mrun : mrun - OFF;
                float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < HC; ++k) {
                    s[k] = full || k < h0 ? as_ex2(fmaf(s[k], qs, -sub)) : 0.f;
                    l4[k & 3] += s[k];
                }
                lsum += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                if (C::KF32) {
                    // weight x 2^(its value row's exponent), relative to the running maximum M
#pragma unroll
                    for (int k = 0; k < HC; k += 2) {
                        const float4 vs = *(const float4*)&m->vsc[j & 3][half * HC + k];
                        // (beyond 2^126 the weight itself is below 2^-112: its share is lost either way)
                        s[k] *= as_ex2(fminf(vs.x + fv, 126.f));
                        s[k + 1] *= as_ex2(fminf(vs.z + fv, 126.f));
                    }
                }
                // P over S: hi planes in the first half of the columns, lo in the second
#pragma unroll
                for (int k = 0; k < HC; k += 16) {
                    uint32_t ph[8], pl[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (C::NQ == 2) as_split(s[k + 2 * i], s[k + 2 * i + 1], ph[i], pl[i]);
                        else ph[i] = as_pack<C::BF>(s[k + 2 * i], s[k + 2 * i + 1]);
                    }
                    as_st8(sb + (half * HC + k) / 2, ph);
                    if (C::NQ == 2) as_st8(sb + KT / 2 + (half * HC + k) / 2, pl);
                }
                as_wait_st();
            }
            as_tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&m->p_full[bf]);
            if (!first) add_o(j - 1);
            cprev = cnew, prev_act = act, prev_any = any;
            if (t + 1 < t1 && (t + 1) / tpg == kvh) continue;

            // ---- the segment's last tile: add it, then the output or a partial
            add_o(j);
            m->lx[half][row] = lsum;
            as_pair_sync(1 + q4);
            float l = lsum + m->lx[half ^ 1][row];
            as_pair_sync(1 + q4);
            if (*(volatile int*)&m->fail) l = NAN;
            if (!live) continue;
            const int d0 = half * HD;
            if (seg_t0 == kvh * tpg && t + 1 == (kvh + 1) * tpg) {
                float inv = l == 0.f ? 0.f : 1.f / l;
                if (C::KF32 && l != 0.f) inv *= exp2f(Mrun - mrun - OFF);
                const size_t at = (size_t)(seq0 + sq) * a.out_sn + (size_t)(kvh * G + row % G) * a.out_sh + d0;
                if constexpr (C::QF32) {
                    float* dst = (float*)a.out + at;
#pragma unroll
                    for (int k = 0; k < HD; k += 4)
                        if (d0 + k < a.hd)
                            *(float4*)(dst + k) = make_float4(o[k] * inv, o[k + 1] * inv, o[k + 2] * inv, o[k + 3] * inv);
                } else {
                    uint16_t* dst = (uint16_t*)a.out + at;
#pragma unroll
                    for (int k = 0; k < HD; k += 8)
                        if (d0 + k < a.hd)
                            *(uint4*)(dst + k) = make_uint4(as_pack<C::BF>(o[k] * inv, o[k + 1] * inv),
                                                            as_pack<C::BF>(o[k + 2] * inv, o[k + 3] * inv),
                                                            as_pack<C::BF>(o[k + 4] * inv, o[k + 5] * inv),
                                                            as_pack<C::BF>(o[k + 6] * inv, o[k + 7] * inv));
                }
            } else {
                // slot 1: a run that began in an earlier kv head; slot 0: the others
                const size_t ps = (size_t)blockIdx.x * 2 + (t0 < kvh * tpg ? 1 : 0);
                if (half == 0) a.part_ml[ps * AS_ROWS + row] = make_float4(mrun, l, C::KF32 ? Mrun - OFF : mrun, 0.f);
                if (mrun != -INFINITY || isnan(l)) {
                    float* dst = a.part_o + (ps * AS_ROWS + row) * 128 + d0;
#pragma unroll
                    for (int k = 0; k < HD; k += 4)
                        if (d0 + k < a.hd) *(float4*)(dst + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
        }
    }
    as_tc_before();
    __syncthreads();
    if (warp == AS_MMA) {
        as_tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
    if (tid == 0 && a.error && *(volatile int*)&m->fail) atomicOr(a.error, 2u);
}

// Adds the partials of a (row tile, kv head) that several CTAs share, in CTA
// order: out = sum O_i 2^(M_i - M) / sum l_i 2^(m_i - m) * 2^(M - m). One warp per row.
template <typename OT, bool KF32>
__global__ void __launch_bounds__(256) k_attn_merge(const __grid_constant__ AttnSharedArgs a, int KT) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int gw = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = gw % AS_ROWS, kvh = gw / AS_ROWS % a.n_kv, rt = gw / AS_ROWS / a.n_kv;
    const int n = a.n_dev ? *a.n_dev : a.n;
    const int prefix = a.prefix_dev ? (int)*a.prefix_dev : a.prefix;
    const int G = a.group, spt = AS_ROWS / G, seq = rt * spt + row / G;
    if (row >= spt * G || seq >= n) return;
    const int tpg = (prefix + KT - 1) / KT + as_suffix_tiles(a, rt * spt, min(spt, n - rt * spt), prefix, KT);
    if (tpg == 0) return;
    const int b0 = a.plan[2 * rt], nb = a.plan[2 * rt + 1], total = tpg * a.n_kv;
    const int g0 = kvh * tpg, g1 = g0 + tpg;
    const int i0 = (int)(((long long)(g0 + 1) * nb - 1) / total), i1 = (int)(((long long)g1 * nb - 1) / total);
    if (as_part(i0, total, nb) <= g0 && as_part(i0 + 1, total, nb) >= g1) return;  // written by its one CTA
    const int nseg = i1 - i0 + 1;
    // lanes take segments: the maxima first
    float m = -INFINITY, M = -INFINITY;
    bool bad = false;
    for (int i = lane; i < nseg; i += 32) {
        const int s0 = as_part(i0 + i, total, nb), s1 = as_part(i0 + i + 1, total, nb);
        if (s0 >= s1) continue;
        const float4 x = a.part_ml[((size_t)(b0 + i0 + i) * 2 + (s0 < g0 ? 1 : 0)) * AS_ROWS + row];
        m = fmaxf(m, x.x), M = fmaxf(M, x.z);
        bad |= isnan(x.y);
    }
    m = warp_max(m), M = warp_max(M);
    bad = __any_sync(0xffffffffu, bad);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool on = 4 * lane < a.hd;
#pragma unroll 4
    for (int i = 0; i < nseg; ++i) {
        const int s0 = as_part(i0 + i, total, nb), s1 = as_part(i0 + i + 1, total, nb);
        if (s0 >= s1) continue;
        const size_t at = ((size_t)(b0 + i0 + i) * 2 + (s0 < g0 ? 1 : 0)) * AS_ROWS + row;
        const float4 x = a.part_ml[at];
        if (x.x == -INFINITY) continue;
        l = fmaf(x.y, exp2f(x.x - m), l);
        if (on) {
            const float4 v = *(const float4*)(a.part_o + at * 128 + 4 * lane);
            const float c = exp2f(x.z - M);
            o.x = fmaf(v.x, c, o.x), o.y = fmaf(v.y, c, o.y), o.z = fmaf(v.z, c, o.z), o.w = fmaf(v.w, c, o.w);
        }
    }
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (KF32 && l != 0.f) inv *= exp2f(M - m);
    if (bad) inv = NAN;
    if (!on) return;
    const size_t at = (size_t)seq * a.out_sn + (size_t)(kvh * G + row % G) * a.out_sh + 4 * lane;
    if constexpr (sizeof(OT) == 4) {
        *(float4*)((float*)a.out + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
        constexpr bool BF = sizeof(OT) == 2 && !__is_same(OT, __half);
        *(uint2*)((uint16_t*)a.out + at) =
            make_uint2(as_pack<BF>(o.x * inv, o.y * inv), as_pack<BF>(o.z * inv, o.w * inv));
    }
}

// ---------------------------------------------------------------- host

static int as_mode(int qt, int kt) {
    if (qt == DT_F32) return kt == DT_F32 ? 0 : kt == DT_F16 ? 1 : -1;
    if (qt == DT_F16 && kt == DT_F16) return 2;
    if (qt == DT_BF16 && kt == DT_BF16) return 3;
    return -1;
}
bool attn_shared_types(int q_type, int kv_type) { return as_mode(q_type, kv_type) >= 0; }

static int as_row_tiles(int n, int group) { return (n + AS_ROWS / group - 1) / (AS_ROWS / group); }
// CTAs of a call: one per SM, at least one per row tile.
static int as_grid(int n, int group, int sms) {
    const int r = as_row_tiles(n, group);
    return r > sms ? r : sms;
}

// Workspace: [2 per CTA][128 rows] (m, l, M), the same rows' O, the row tiles' plan.
size_t attn_shared_work_bytes(int n, int group, int sms) {
    const size_t cta = as_grid(n, group, sms);
    return cta * 2 * AS_ROWS * (16 + 128 * 4) + (size_t)as_row_tiles(n, group) * 8 + 256;
}

template <int MODE, int DP>
static cudaError_t as_launch(AttnSharedArgs a, int sms, cudaStream_t s) {
    using C = AsCfg<MODE, DP>;
    const int R = as_row_tiles(a.n, a.group), spt = AS_ROWS / a.group;
    // Few tiles per (row tile, kv head): one CTA each, and no partials to add. A
    // tile takes a CTA about 2 us with its latencies, the second kernel about 3.
    const long long most = (a.prefix + C::KT - 1) / C::KT +
                           (long long)(a.n < spt ? a.n : spt) * ((a.slot_len + C::KT - 1) / C::KT);
    a.whole = !a.prefix_dev && most <= 3 && (long long)R * a.n_kv <= 0x7fffffff;
    const int grid = a.whole ? R * a.n_kv : as_grid(a.n, a.group, sms);
    k_attn_shared<MODE, DP><<<grid, AS_THREADS, C::SMEM, s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || a.whole) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * a.n_kv * (AS_ROWS / 8)));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    using OT = typename std::conditional<MODE <= 1, float,
                                         typename std::conditional<MODE == 2, __half, __nv_bfloat16>::type>::type;
    return cudaLaunchKernelEx(&cfg, k_attn_merge<OT, MODE == 0>, a, (int)C::KT);
}

cudaError_t launch_attn_shared(AttnSharedArgs a, int q_type, int kv_type, void* work, int sms, cudaStream_t s) {
    const size_t cta = as_grid(a.n, a.group, sms);
    a.part_ml = (float4*)work;
    a.part_o = (float*)((uint8_t*)work + cta * 2 * AS_ROWS * 16);
    a.plan = (int*)((uint8_t*)work + cta * 2 * AS_ROWS * (16 + 128 * 4));
    const bool wide = a.hd > 64;
    switch (as_mode(q_type, kv_type)) {
        case 0: return wide ? as_launch<0, 128>(a, sms, s) : as_launch<0, 64>(a, sms, s);
        case 1: return wide ? as_launch<1, 128>(a, sms, s) : as_launch<1, 64>(a, sms, s);
        case 2: return wide ? as_launch<2, 128>(a, sms, s) : as_launch<2, 64>(a, sms, s);
        case 3: return wide ? as_launch<3, 128>(a, sms, s) : as_launch<3, 64>(a, sms, s);
    }
    return cudaErrorInvalidValue;
}

template <int MODE, int DP>
static cudaError_t as_configure() {
    return cudaFuncSetAttribute(k_attn_shared<MODE, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                AsCfg<MODE, DP>::SMEM);
}
cudaError_t attn_shared_configure() {
    cudaError_t e = as_configure<0, 64>();
    if (e == cudaSuccess) e = as_configure<0, 128>();
    if (e == cudaSuccess) e = as_configure<1, 64>();
    if (e == cudaSuccess) e = as_configure<1, 128>();
    if (e == cudaSuccess) e = as_configure<2, 64>();
    if (e == cudaSuccess) e = as_configure<2, 128>();
    if (e == cudaSuccess) e = as_configure<3, 64>();
    if (e == cudaSuccess) e = as_configure<3, 128>();
    return e;
}

}  // namespace talos
