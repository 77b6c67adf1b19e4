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
// to an integer (base 2), so every rescaling is by an exact power of two. For f32
// outputs O is added up in registers (the tensor core only sums one tile: its
// accumulation truncates); for 16-bit outputs it stays in tensor memory for runs of
// AS_RUN prefix tiles. A step of 16 keys was seen to lose 2 to 3 units in the last
// place of the sum, always towards zero: with one run over 2,048 tiles the output was
// 1.5e-3 to 2e-3 too small; a run of 16 loses about 1.5e-5 (half a step of f16 is 2.4e-4).
//
// Precision. f16 / bf16 queries: one product each, P rounded to 16 bits (half a
// step of 2^-11 / 2^-8 relative per weight, averaged by the sum; the row's sum is that
// of the rounded weights), f32 everywhere else. f32 queries: q is scaled by a power
// of two into [2^14, 2^15) at its row's largest element and split into f16 hi + lo
// (22 bits), and so is P. An f32 cache's tiles are scaled (one power of two for 64
// keys of K, and of V) and split too, so no input overflows f16; an element keeps
// 22 bits, or 2^-39 of its tile's largest where that is more. lo x lo (2^-22) is
// left out.
//
// Roles (one CTA per SM):
//  * warps 0-7: softmax. Warps w and w + 4 share the rows 32 w .. 32 w + 31 (their
//    TMEM lanes), one half of the tile's keys and of the head's dims each; they
//    exchange row maxima in shared memory. f32 queries come as they are; these warps
//    scale and split them into tensor memory (as an operand from shared memory Q
//    would be read again for every product: 6 KB instead of 2 per 128 x 64 x 16).
//  * 16-bit caches, 12 warps: warp 8 issues the TMA copies of the K tiles and the
//    queries, warp 9 those of the V tiles, straight into the swizzled operand tiles
//    (separate, so that K runs ahead of V).
//  * f32 cache, 20 warps: warp 17 fills a ring of 16 KB slots by TMA (the queries of a
//    kv head, then half tiles, or whole ones of heads up to 64); warps 8-11 scale and
//    split the K tiles into the operand tiles, warps 12-15 the V tiles (side by side:
//    a tile takes either about 4,500 clocks, most of them latencies).
//  * the last two warps issue the MMAs: the last one (which allocates TMEM) S = Q K^T,
//    a tile ahead of the other's O = P V, so that the softmax of one tile runs beside
//    the products of its neighbours. Tiles that end early take fewer of both. The
//    copies bring along the rows behind a suffix's last key, which may hold anything:
//    the PV warp clears those V rows that its product reads.
// Bound: the latencies between the roles of the one CTA an SM. Measured: 64 sequences,
// 64 / 8 heads of 128, bf16, 32768 shared and up to 1024 own positions 155-162 us, 0.44
// PFLOP/s (2,300 clocks a dense tile; its exponentials and its products would take 1,024
// each, side by side); 32 sequences, f32 queries and f16 cache, 8192 and up to 512, 43-48
// us, 1.5 TB/s of keys once (suffix tiles: from S to O); 32 sequences, 32 / 8 heads, f32,
// 1024 and up to 256, 33-35 us (the f32 tiles' conversion).
//
// Every wait is bounded; on expiry a CTA flag makes all roles run on without
// waiting or multiplying, and the rows come out as NaN.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "ops.cuh"
#include "ptx.cuh"

namespace talos {

constexpr int AS_ROWS = 128;   // rows per tile = TMEM lanes
constexpr int AS_SOFT = 8;     // softmax warps
constexpr int AS_CONV = 4;     // f32: converter warps of K, and of V
constexpr int AS_SLOT = 16 * 1024;  // f32: one slot of the ring
constexpr int AS_MISC = 12 * 1024;
constexpr int AS_SMEM = 227 * 1024;
constexpr int AS_RUN = 16;  // 16-bit outputs: prefix tiles added up in tensor memory
constexpr float AS_LOG2E = 1.4426950408889634f;

// MODE: types of (q, cache): 0 (f32, f32), 1 (f32, f16), 2 (f16, f16), 3 (bf16, bf16)
template <int MODE, int DP>
struct AsCfg {
    static constexpr bool QF32 = MODE <= 1, KF32 = MODE == 0, BF = MODE == 3;
    static constexpr int NQ = QF32 ? 2 : 1;  // planes (hi, lo) of Q
    static constexpr int NP = QF32 ? 2 : 1;  // of P
    static constexpr int NK = KF32 ? 2 : 1;  // of K and V
    static constexpr int KT = KF32 ? 64 : 128;   // keys per tile
    static constexpr int WARPS = KF32 ? 20 : 12;
    static constexpr int THREADS = WARPS * 32;   // x 96 or 168 registers at launch
    // registers after the split: 256 x 152 + 384 x 56 <= 640 x 96, 256 x 208 + 128 x 88 = 384 x 168
    static constexpr int SOFT_REGS = KF32 ? 152 : 208, REST_REGS = KF32 ? 56 : 88;
    static constexpr int Q_BYTES = AS_ROWS * DP * (QF32 ? 4 : 2), KPLANE = KT * DP * 2;
    static constexpr int HALF = AS_SLOT / (DP * 4);  // f32: rows of a ring slot, 32 or 64
    static constexpr int NR = KF32 ? 7 : 0;
    static constexpr int QB = Q_BYTES / AS_SLOT;     // f32: slots of the queries
    // 16-bit outputs: the prefix's O is added up in tensor memory, in O buffer 0. The
    // rows' warps add it to their registers after every AS_RUN tiles and before their
    // suffix tiles, whose products go to buffers 1, 0, 1, ... and are added in registers
    // too: no other row meets their values
    static constexpr bool ACC = !QF32;
    static constexpr int Q_OWN = KF32 ? 0 : Q_BYTES;  // (f32: in the ring)
    static constexpr int FIT = (AS_SMEM - AS_MISC - Q_OWN) / KPLANE;  // 16-bit: operand tiles that fit
    static constexpr int NSV = KF32 ? 2 : (FIT / 2 > 4 ? 4 : FIT / 2);
    static constexpr int NSK = KF32 ? 1 : (FIT - NSV > 4 ? 4 : FIT - NSV);
    static constexpr int SMEM = Q_OWN + (NSK + NSV) * NK * KPLANE + NR * AS_SLOT + AS_MISC;
    static constexpr int S_COLS = KT;          // TMEM columns of one S buffer; P lies over it
    static constexpr int O_COL = 2 * KT;       // first column of the O buffers
    static constexpr int NOB = MODE == 1 ? 1 : 2;
    static constexpr int Q_COL = O_COL + NOB * DP;  // f32 queries: hi, then lo
    static_assert(NSV >= 1 && SMEM <= AS_SMEM, "shared memory");
    static_assert(Q_COL + (QF32 ? DP : 0) <= 512, "tensor memory");
};

struct AsMisc {
    uint64_t q_raw[2], q_full, q_empty[2], k_full[4], k_empty[4], v_full[4], v_empty[4], r_full[8], r_empty[8];
    uint64_t s_full[2], p_full[2], o_full[2], o_empty[2], done;
    uint32_t tmem;
    int fail;
    uint32_t q_slot[2], q_par[2];  // f32: the first ring slot of the queries, its parity (two segments in flight at most)
    int rt, b0, nb, tpg;     // row tile of this CTA, its first CTA and CTA count, tiles per kv head
    int cum[AS_ROWS + 1];    // suffix tiles before each of the row tile's sequences
    int len[AS_ROWS], slot[AS_ROWS];
    float mx[2][2][AS_ROWS];  // [tile parity][half] row maxima
    float lx[2][AS_ROWS];
    float ksc[4], vsc[4];     // f32 cache: 2^exponent of a tile's keys, values
    uint32_t cmax[2][2][AS_CONV];  // f32 cache: largest |element| of each converter warp (K, V; tile parity)
};
static_assert(sizeof(AsMisc) <= AS_MISC, "misc area");

// The tensor maps of a call (CUtensorMap): queries (16-bit), the prefix's and the slots' rows.
struct AsMaps {
    CUtensorMap q, kp, vp, k, v;
};

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
__device__ __forceinline__ bool as_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void as_tma3(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void as_tma4(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                        uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
// two f32 in a 64-bit register pair
typedef unsigned long long f2;
__device__ __forceinline__ f2 as_f2(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void as_un2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 as_fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 as_add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 as_mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float as_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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
// The same split of a pair whose hi keeps 10 mantissa bits by truncation (exact in
// f16 for |x| in its normal range; below it both parts round): fewer conversions.
__device__ __forceinline__ void as_split_cut(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ha = __uint_as_float(__float_as_uint(a) & 0xffffe000u), hb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
    hi = as_pack<false>(ha, hb);
    lo = as_pack<false>(a - ha, b - hb);
}
// The exponent e of the largest |x| (its bits), as used for scaling: x 2^(14 - e)
// lies in [2^14, 2^15); kept where 2^(14 - e) and 2^(e - 14) are normal.
__device__ __forceinline__ int as_exponent(uint32_t abs_bits) {
    const int e = (int)(abs_bits >> 23) - 127;
    return e < -112 ? -112 : e;
}
__device__ __forceinline__ float as_pow2(int e) { return __int_as_float((e + 127) << 23); }

// Bounded wait (4 M polls, each of which the hardware suspends for a while: a
// second or so). On expiry it marks the CTA as failed and `ok` as false: the role
// then runs its loops to their end without waiting, copying, multiplying or
// signalling (the pair barriers still match), and the others follow when their own
// waits find the mark. Kept small: it is inlined some thirty times, and what runs
// in the roles' loops has to stay near in the instruction caches.
__device__ __forceinline__ void as_wait(AsMisc* m, uint64_t* bar, uint32_t parity, bool& ok) {
    if (!ok) return;
    uint32_t polls = 0;
    while (!mbar_try_wait(bar, parity)) {
        if (++polls & 4095) continue;
        if (polls >= 1u << 22 || *(volatile int*)&m->fail) {
            *(volatile int*)&m->fail = 1;
            ok = false;
            break;
        }
    }
}
__device__ __forceinline__ void as_arrive(uint64_t* bar, bool ok) {
    if (ok) mbar_arrive(bar);
}
// After a failure: time for the copies that a role has in flight to land.
__device__ __forceinline__ void as_settle(bool ok) {
    if (ok) return;
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
}

// First tile of part i of n tiles cut into nb even parts (the first n % nb parts
// are one longer), and the part that holds tile x.
__device__ __forceinline__ int as_part(int i, int n, int nb) {
    const int q = n / nb, r = n - q * nb;
    return i * q + min(i, r);
}
__device__ __forceinline__ int as_part_of(int x, int n, int nb) {
    const int q = n / nb, r = n - q * nb, cut = r * (q + 1);
    return x < cut ? x / (q + 1) : r + (x - cut) / max(q, 1);
}

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

// A role's walk over its CTA's tiles: tile `off` of kv head `kvh`; its first key (of
// the prefix, or of sequence i's suffix) and the number of its keys.
struct AsWalk {
    int off, kvh, i, key, valid;
    __device__ __forceinline__ void start(int t0, int tpg) {
        kvh = t0 / tpg, off = t0 - kvh * tpg, i = 0;
    }
    __device__ __forceinline__ void tile(const AsMisc* m, int ntp, int prefix, int KT) {
        if (off < ntp) {
            key = off * KT;
            valid = min(KT, prefix - key);
        } else {
            while (m->cum[i + 1] <= off - ntp) ++i;  // (past sequences without a suffix)
            key = (off - ntp - m->cum[i]) * KT;
            valid = min(KT, m->len[i] - key);
        }
    }
    __device__ __forceinline__ void next(int tpg) {
        if (++off == tpg) off = 0, ++kvh, i = 0;
    }
};
// Suffix tiles of sequences seq0 .. seq0 + ns - 1, summed by a warp.
__device__ __forceinline__ int as_suffix_tiles(const AttnSharedArgs& a, int seq0, int ns, int prefix, int KT) {
    int t = 0;
    for (int i = threadIdx.x & 31; i < ns; i += 32)
        if (as_slot(a, seq0 + i) >= 0) t += (as_len(a, seq0 + i, prefix) + KT - 1) / KT;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// f32 tiles: NW warps read the rows of a raw tile (two ring slots of HALF rows, or
// one) for the largest element, then again and store the tile scaled by 2^(14 - e) as
// f16 hi and lo operand tiles. Rows behind the last key (the next ones of the slot, or
// stale) become zeros.
template <int DP, int KT, int NW>
struct AsConv {
    static constexpr int QC = DP / 4, QR = 32 / QC;  // float4 chunks of a row, rows per warp step
    static constexpr int NI = KT / QR / NW, HALF = AS_SLOT / (DP * 4);
    static_assert(NI * QR * NW == KT, "rows of a warp");
    static __device__ __forceinline__ float4 chunk(const uint8_t* raw0, const uint8_t* raw1, int r, int ch, int valid) {
        if (r >= valid) return make_float4(0.f, 0.f, 0.f, 0.f);
        return *(const float4*)((r < HALF ? raw0 : raw1) + r % HALF * (QC * 16) + ch * 16);
    }
    // the warp's largest finite |element| as bits (an infinite one must not scale the others to 0)
    static __device__ __forceinline__ uint32_t largest(const uint8_t* raw0, const uint8_t* raw1, int w, int lane,
                                                       int valid) {
        const int ch = lane % QC, sub = lane / QC;
        float mx = 0.f;
#pragma unroll 8
        for (int q = 0; q < NI; ++q) {
            const float4 v = chunk(raw0, raw1, (w + NW * q) * QR + sub, ch, valid);
            mx = as_max3(mx, fabsf(v.x), fabsf(v.y));
            mx = as_max3(mx, fabsf(v.z), fabsf(v.w));
        }
        uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
        if (top == 0x7f800000u) {
            mx = 0.f;
#pragma unroll 1
            for (int q = 0; q < NI; ++q) {
                const float4 v = chunk(raw0, raw1, (w + NW * q) * QR + sub, ch, valid);
                for (const float x : {v.x, v.y, v.z, v.w})
                    if (fabsf(x) < INFINITY) mx = fmaxf(mx, fabsf(x));
            }
            top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
        }
        return top;
    }
    static __device__ __forceinline__ void store(const uint8_t* raw0, const uint8_t* raw1, uint8_t* tile, int w, int lane,
                                                 int valid, int e) {
        const int ch = lane % QC, sub = lane / QC;
        const float f = as_pow2(14 - e);
        const f2 ff = as_f2(f, f);
        uint8_t* dst0 = tile + (ch / 16) * (KT * 128) + (ch & 1) * 8;
#pragma unroll 8
        for (int q = 0; q < NI; ++q) {
            const int r = (w + NW * q) * QR + sub;
            const float4 v = chunk(raw0, raw1, r, ch, valid);
            float x, y, z, u;
            as_un2(as_mul2(as_f2(v.x, v.y), ff), x, y), as_un2(as_mul2(as_f2(v.z, v.w), ff), z, u);
            uint2 hi, lo;
            as_split_cut(x, y, hi.x, lo.x);
            as_split_cut(z, u, hi.y, lo.y);
            uint8_t* dst = dst0 + r * 128 + (((ch % 16 / 2) ^ (r & 7)) << 4);
            *(uint2*)dst = hi;
            *(uint2*)(dst + KT * DP * 2) = lo;
        }
        as_fence_async();
        __syncwarp();
    }
};

// ---------------------------------------------------------------- the kernel

template <int MODE, int DP>
__global__ void __launch_bounds__((AsCfg<MODE, DP>::THREADS), 1)
    k_attn_shared(const __grid_constant__ AttnSharedArgs a, const __grid_constant__ AsMaps maps) {
    using C = AsCfg<MODE, DP>;
    constexpr int KT = C::KT, NB = DP / 64;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;                              // f32 queries: [DP / 32][128 rows][32], else the operand
    uint8_t* sK = sQ + C::Q_OWN;            // [NSK][planes]
    uint8_t* sV = sK + C::NSK * C::NK * C::KPLANE;   // [NSV][planes]
    uint8_t* sR = sV + C::NSV * C::NK * C::KPLANE;   // f32: [NR] ring slots
    AsMisc* m = (AsMisc*)(sR + C::NR * AS_SLOT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    const int n = a.n_dev ? *a.n_dev : a.n;
    const int prefix = a.prefix_dev ? (int)*a.prefix_dev : a.prefix;
    const int G = a.group, spt = AS_ROWS / G;          // sequences per row tile
    const int R = (n + spt - 1) / spt;
    const int ntp = (prefix + KT - 1) / KT;

    // ---- set-up: barriers, TMEM, this CTA's row tile and its run of tiles
    // (the parameters' lines are read here together: one miss instead of one after another)
    asm volatile("" ::"l"(a.q), "l"(a.kp), "l"(a.k), "l"(a.slot_sh), "l"(a.out), "r"(a.hd), "l"(a.lens), "l"(a.n_dev),
                 "l"(a.part_o));
    if (warp == C::WARPS - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&m->tmem)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid >= 96 && tid < 101) {  // the call's tensor maps (those that it has)
        const int i = tid - 96;
        if (i == 0 || (i < 3 ? a.prefix > 0 : a.slot_len > 0))
            asm volatile("prefetch.tensormap [%0];" ::"l"((const CUtensorMap*)&maps + i) : "memory");
    }
    if (tid == 64) {
        m->fail = 0;
        mbar_init(&m->q_full, C::QF32 ? AS_SOFT : 1);
        mbar_init(&m->q_raw[0], 1);
        mbar_init(&m->q_raw[1], 1);
        // (one for the even kv heads of a run and one for the odd: with heads up to 64 the softmax
        // warps can be done with a kv head's queries before the copies wait for those before)
        mbar_init(&m->q_empty[0], C::QF32 ? AS_SOFT : 1);
        mbar_init(&m->q_empty[1], C::QF32 ? AS_SOFT : 1);
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            mbar_init(&m->k_full[i], C::KF32 ? AS_CONV : 1);
            mbar_init(&m->k_empty[i], 1);
            mbar_init(&m->v_full[i], C::KF32 ? AS_CONV : 1);
            mbar_init(&m->v_empty[i], 1);
        }
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            mbar_init(&m->r_full[i], 1);
            mbar_init(&m->r_empty[i], AS_CONV);
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            mbar_init(&m->s_full[i], 1);
            mbar_init(&m->p_full[i], AS_SOFT);
            mbar_init(&m->o_full[i], 1);
            mbar_init(&m->o_empty[i], AS_SOFT);
        }
        mbar_init(&m->done, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    int rt = 0, b0 = 0, nb = (int)gridDim.x;
    if (a.whole) {  // one CTA per (row tile, kv head)
        rt = (int)blockIdx.x / a.n_kv, b0 = rt * a.n_kv, nb = a.n_kv;
    } else if (R > 1) {
        // CTAs in proportion to the row tiles' work: row tile r has CTAs b(r) ..
        // b(r + 1) - 1, b(r) = r + (N - R) * (tiles before r) / (all tiles)
        int* cnt = (int*)smem;  // [R] suffix tiles, before the operand tiles are used
        for (int r = warp; r < R; r += C::WARPS) {
            const int own = as_suffix_tiles(a, r * spt, min(spt, n - r * spt), prefix, KT);
            if (lane == 0) cnt[r] = own;
        }
        __syncthreads();
        if (warp == 0) {
            const int N = gridDim.x;
            int total = 0, before = 0;  // tiles of one kv head
            for (int r = lane; r < R; r += 32) total += ntp + cnt[r];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            const double per = total ? (double)(N - R) / (double)total : 0.0;
            if (lane == 0) m->rt = -1;
            __syncwarp();
            for (int r0 = 0; r0 < R; r0 += 32) {
                const int r = r0 + lane;
                const int t = r < R ? ntp + cnt[r] : 0;
                int x = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                const int lo = r + (int)(per * (double)(before + x - t)), hi = r + 1 + (int)(per * (double)(before + x));
                if (r < R) {
                    if ((int)blockIdx.x >= lo && (int)blockIdx.x < hi) m->rt = r, m->b0 = lo, m->nb = hi - lo;
                }
                before += __shfl_sync(0xffffffffu, x, 31);
            }
        }
        as_fence_async();  // (cnt's bytes are written by TMA copies next)
        __syncthreads();
        rt = m->rt, b0 = m->b0, nb = m->nb;
    }
    const bool mine = rt >= 0 && rt < R;
    const int seq0 = mine ? rt * spt : 0, nseq = mine ? min(spt, n - seq0) : 0;
    if (warp == 0) {  // the row tile's suffix list
        int run = 0;
        for (int i0 = 0; i0 < nseq; i0 += 32) {
            const int i = i0 + lane;
            int slot = -1, len = 0;
            if (i < nseq) {
                slot = as_slot(a, seq0 + i);
                len = as_len(a, seq0 + i, prefix);
                if (slot < 0) len = 0;
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
    as_tc_before();
    __syncthreads();
    as_tc_after();
    const uint32_t tmem = m->tmem;
    const int tpg = m->tpg, total = tpg * a.n_kv;  // tiles per kv head, tiles of the row tile
    const int rank = (int)blockIdx.x - b0;
    const int t0 = mine ? as_part(rank, total, nb) : 0, t1 = mine ? as_part(rank + 1, total, nb) : 0;
    const int rows = nseq * G;  // live rows
    if (mine && rank == 0 && tid == 0 && !a.whole)
        a.plan[3 * rt] = b0, a.plan[3 * rt + 1] = nb, a.plan[3 * rt + 2] = tpg;  // for k_attn_merge
    if (mine && tpg == 0 && rank == 0) {
        // no key in the whole row tile: zeros
        for (int i = tid; i < rows * a.n_kv * a.hd; i += C::THREADS) {
            const int d = i % a.hd, h = i / a.hd % (G * a.n_kv), sq = seq0 + i / a.hd / (G * a.n_kv);
            const size_t at = (size_t)sq * a.out_sn + (size_t)h * a.out_sh + d;
            if (C::QF32) ((float*)a.out)[at] = 0.f;
            else ((uint16_t*)a.out)[at] = 0;
        }
    }
    auto ring_step = [&](uint32_t& st, uint32_t& par, uint32_t by) {  // f32: on by up to NR slots
        st += by;
        if (st >= (uint32_t)(C::NR ? C::NR : 1)) st -= C::NR, par ^= 1;
    };
    bool ok = true;
    // the queries of kv head kvh: their live rows, 128 bytes of each at a time
    auto copy_q = [&](int kvh, int seg) {
        constexpr int W = C::QF32 ? 32 : 64;
        uint64_t* bar = C::QF32 ? &m->q_raw[seg & 1] : &m->q_full;
        if (seg > 0) as_wait(m, &m->q_empty[(seg - 1) & 1], ((seg - 1) >> 1) & 1, ok);
        if (!ok) return;
        mbar_expect_tx(bar, (uint32_t)(min(spt, a.n) * G) * 128 * (DP / W));
#pragma unroll
        for (int b = 0; b < DP / W; ++b)
            as_tma3(smem_u32(sQ) + b * (AS_ROWS * 128), &maps.q, W * b, kvh * G, seq0, bar);
    };
    if (t0 >= t1) {
        // nothing to do (TMEM is freed below)
    } else if (warp >= AS_SOFT) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REST_REGS));
    if (warp == C::WARPS - 1) {
        // ---------------------------------------------------- S = Q K^T: the warp walks the tiles
        // together (uniform control flow and descriptors), one lane issues
        const bool lead = as_elect();
        const int ksteps = (a.hd + 15) / 16;
        const uint64_t dq = as_desc(smem_u32(sQ), 16), dk0 = as_desc(smem_u32(sK), 16);
        int j = 0, seg = -1, cur = -1;
        uint32_t sk = 0, pk = 0;  // stage and its parity
        AsWalk w;
        w.start(t0, tpg);
        for (int t = t0; t < t1; ++t, ++j) {
            if (w.kvh != cur) {
                cur = w.kvh, ++seg;
                as_wait(m, &m->q_full, seg & 1, ok);
            }
            const uint32_t bf = j & 1;
            w.tile(m, ntp, prefix, KT);
            const uint32_t idesc = as_idesc((w.valid + 15) & ~15, C::BF, false);
            as_wait(m, &m->k_full[sk], pk, ok);
            if (j >= 2) as_wait(m, &m->o_full[bf], ((j - 2) >> 1) & 1, ok);  // P over this S buffer was read
            as_tc_after();
            if (lead && ok) {
                const uint32_t d = tmem + bf * C::S_COLS;
                const uint64_t k = dk0 + (uint64_t)(sk * (C::NK * C::KPLANE >> 4));
                // the small terms first
#pragma unroll
                for (int pr = C::NQ + C::NK - 2; pr >= 0; --pr) {
                    const bool ql = C::NQ == 2 && pr == 1, kl = pr == 2;
                    const uint32_t first = pr == C::NQ + C::NK - 2 ? 0u : 1u;
                    const uint64_t kd = k + (kl ? C::KPLANE >> 4 : 0);
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ++ks) {
                        if (ks >= ksteps) continue;
                        const uint64_t ka = kd + (uint64_t)(((ks >> 2) * (KT * 128) + (ks & 3) * 32) >> 4);
                        if (C::QF32)
                            as_mma_ts(d, tmem + C::Q_COL + (ql ? DP / 2 : 0) + 8 * ks, ka, idesc, ks ? 1u : first);
                        else
                            as_mma_ss(d, dq + (uint64_t)(((ks >> 2) * (AS_ROWS * 128) + (ks & 3) * 32) >> 4), ka, idesc,
                                      ks ? 1u : first);
                    }
                }
                as_commit(&m->k_empty[sk]);
                as_commit(&m->s_full[bf]);
                if (!C::QF32 && (t + 1 == t1 || w.off + 1 == tpg)) as_commit(&m->q_empty[seg & 1]);  // the queries may be replaced
            }
            __syncwarp();
            w.next(tpg);
            if (++sk == C::NSK) sk = 0, pk ^= 1;
        }
        // nothing in flight when TMEM is freed (also after a failure: a wait of its own)
        if (lead) as_commit(&m->done);
        bool end_ok = true;
        as_wait(m, &m->done, 0, end_ok);
    } else if (warp == C::WARPS - 2) {
        // ---------------------------------------------------- O = P V
        const bool lead = as_elect();
        const uint32_t idesc = as_idesc((a.hd + 15) / 16 * 16, C::BF, true);
        const uint64_t dv0 = as_desc(smem_u32(sV), KT * 128);
        int j = 0, cur = -1, seg_t0 = t0, nsuf = 0, ntaken = 0;  // ACC: suffix tiles of the segment, hand-overs before it
        uint32_t sv = 0, pv = 0;
        AsWalk w;
        w.start(t0, tpg);
        for (int t = t0; t < t1; ++t, ++j) {
            const uint32_t bf = j & 1, par = (j >> 1) & 1;
            const bool pre = w.off < ntp, pre0 = w.kvh != cur;
            cur = w.kvh;
            if (pre0) seg_t0 = t;
            w.tile(m, ntp, prefix, KT);
            const int valid = w.valid, ksteps = (valid + 15) / 16;
            as_wait(m, &m->v_full[sv], pv, ok);
            if (!C::KF32 && !pre && (valid & 15)) {
                uint8_t* v = sV + sv * C::KPLANE;
                for (int c = valid * 8 + lane; c < ksteps * 128; c += 32)
#pragma unroll
                    for (int b = 0; b < NB; ++b) *(uint4*)(v + b * (KT * 128) + c * 16) = make_uint4(0, 0, 0, 0);
                as_fence_async();
                __syncwarp();
            }
            // the O buffer is free: two in turn, one for all, or (ACC) one for the suffix tiles
            if (C::ACC) {
                // hand-overs of a buffer, counted over the CTA: the prefix's O, then each suffix
                // tile's; suffix tile k of a segment waits for hand-over k - 1
                if (pre0) ntaken += nsuf ? nsuf + 1 : 0, nsuf = 0;
                if (!pre && nsuf > 0) {
                    const int h = ntaken + nsuf - 1;
                    as_wait(m, &m->o_empty[h & 1], (h >> 1) & 1, ok);
                }
            } else if (C::NOB == 2) {
                as_wait(m, &m->o_empty[bf], par ^ 1, ok);
            } else if (j > 0) {
                as_wait(m, &m->o_empty[0], (j - 1) & 1, ok);
            }
            as_wait(m, &m->p_full[bf], par, ok);
            as_tc_after();
            if (lead && ok) {
                const uint32_t d = tmem + C::O_COL + (C::ACC ? (pre ? 0 : (nsuf & 1) ^ 1) : C::NOB == 2 ? bf : 0) * DP, p = tmem + bf * C::S_COLS;
                const uint32_t keep = C::ACC && pre && (t - seg_t0) % AS_RUN ? 1u : 0u;
                const uint64_t v = dv0 + (uint64_t)(sv * (C::NK * C::KPLANE >> 4));
                // the small terms first
#pragma unroll
                for (int pr = C::NP + C::NK - 2; pr >= 0; --pr) {
                    const bool p_lo = C::NP == 2 && pr == 1, v_lo = pr == 2;
                    const uint32_t pa = p + (p_lo ? KT / 2 : 0), first = pr == C::NP + C::NK - 2 ? keep : 1u;
                    const uint64_t vd = v + (v_lo ? C::KPLANE >> 4 : 0);
#pragma unroll
                    for (int ks = 0; ks < KT / 16; ++ks) {
                        if (ks >= ksteps) continue;
                        as_mma_ts(d, pa + 8 * ks, vd + (uint64_t)(ks * 2048 >> 4), idesc, ks ? 1u : first);
                    }
                }
                as_commit(&m->v_empty[sv]);
                as_commit(&m->o_full[bf]);
            }
            if (C::ACC) nsuf += !pre;
            __syncwarp();
            w.next(tpg);
            if (++sv == C::NSV) sv = 0, pv ^= 1;
        }
        if (lead) as_commit(&m->done);
    } else if (!C::KF32 && (warp == 8 || warp == 9)) {
        // ---------------------------------------------------- TMA: K (and 16-bit queries), V
        if (as_elect()) {
            const bool is_v = warp == 9;
            const CUtensorMap *mp = is_v ? &maps.vp : &maps.kp, *ms = is_v ? &maps.v : &maps.k;
            uint64_t *full = is_v ? m->v_full : m->k_full, *empty = is_v ? m->v_empty : m->k_empty;
            const uint32_t ns = is_v ? C::NSV : C::NSK;
            const uint32_t base = smem_u32(is_v ? sV : sK);
            uint32_t st = 0, par = 1;
            int seg = -1, cur = -1;
            AsWalk w;
            w.start(t0, tpg);
            for (int t = t0; t < t1; ++t) {
                w.tile(m, ntp, prefix, KT);
                as_wait(m, &empty[st], par, ok);
                if (ok) {
                    mbar_expect_tx(&full[st], C::KPLANE);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t dst = base + st * C::KPLANE + b * (KT * 128);
                        if (w.off < ntp) as_tma3(dst, mp, 64 * b, w.kvh, w.key, &full[st]);
                        else as_tma4(dst, ms, 64 * b, w.kvh, w.key, m->slot[w.i], &full[st]);
                    }
                }
                if (!is_v && w.kvh != cur) cur = w.kvh, copy_q(w.kvh, ++seg);
                if (++st == ns) st = 0, par ^= 1;
                w.next(tpg);
            }
            as_settle(ok);
        }
        __syncwarp();
    } else if (C::KF32 && warp == 17) {
        // ---------------------------------------------------- f32: the ring's copies
        if (as_elect()) {
            uint32_t st = 0, par = 0;            // the next slot, the parity of its data
            uint32_t used = 0, re_par = 0;       // bit s: slot s held a tile before; parity of r_empty[s]
            uint32_t held_q = 0, first_q = 0;    // bit s: it held queries (the first of them)
            int seg = -1, cur = -1, q_done = 0;
            auto slot_free = [&]() {
                const uint32_t b = 1u << st;
                if (held_q & b) {
                    if (first_q & b) {
                        as_wait(m, &m->q_empty[q_done & 1], q_done >> 1 & 1, ok);
                        ++q_done;
                    }
                    held_q &= ~b, first_q &= ~b;
                } else if (used & b) {
                    as_wait(m, &m->r_empty[st], re_par >> st & 1, ok);
                    re_par ^= b;
                }
                used |= b;
            };
            auto next = [&]() {
                if (++st == (uint32_t)C::NR) st = 0, par ^= 1;
            };
            AsWalk w;
            w.start(t0, tpg);
            for (int t = t0; t < t1; ++t) {
                if (w.kvh != cur) {  // the queries of a kv head, 32 dims per slot
                    cur = w.kvh, ++seg;
#pragma unroll 1
                    for (int b = 0; b < C::QB; ++b) {
                        slot_free();
                        if (b == 0) {
                            m->q_slot[seg & 1] = st, m->q_par[seg & 1] = par;
                            as_arrive(&m->q_raw[seg & 1], ok);
                            first_q |= 1u << st;
                        }
                        held_q |= 1u << st;
                        if (ok) {
                            mbar_expect_tx(&m->r_full[st], (uint32_t)(min(spt, a.n) * G) * 128);
                            as_tma3(smem_u32(sR) + st * AS_SLOT, &maps.q, 32 * b, w.kvh * G, seq0, &m->r_full[st]);
                        }
                        next();
                    }
                }
                w.tile(m, ntp, prefix, KT);
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {  // K, then V: one or two slots each, both on the first one's barrier
                    const bool two = C::HALF < w.valid;
                    if ((h & 1) && !two) continue;
                    const uint32_t bar_st = (h & 1) ? (st == 0 ? C::NR : st) - 1 : st;
                    slot_free();
                    if (ok) {
                        if (h & 1) mbar_arrive(&m->r_full[st]);  // (its phases count the laps)
                        else mbar_expect_tx(&m->r_full[st], two ? 2 * AS_SLOT : AS_SLOT);
                        uint64_t* bar = &m->r_full[bar_st];
                        const uint32_t dst = smem_u32(sR) + st * AS_SLOT;
                        const int row = w.key + (h & 1) * C::HALF;
                        if (w.off < ntp) as_tma3(dst, h < 2 ? &maps.kp : &maps.vp, 0, w.kvh, row, bar);
                        else
                            as_tma4(dst, h < 2 ? &maps.k : &maps.v, 0, w.kvh, row + a.slot_row0 * prefix, m->slot[w.i],
                                    bar);
                    }
                    next();
                }
                w.next(tpg);
            }
            as_settle(ok);
        }
        __syncwarp();
    } else if constexpr (C::KF32) {
        // ---------------------------------------------------- ring -> operand tiles: K by the first
        // four warps, V by the next (warp 16 only fills up the warpgroup)
        if (warp < 8 + 2 * AS_CONV) {
        const int w = warp & 3;
        const bool is_v = warp >= 8 + AS_CONV;
        int cur = -1, j = 0;
        uint32_t st = 0, par = 0;
        using cv = AsConv<DP, KT, AS_CONV>;
        AsWalk wk;
        wk.start(t0, tpg);
        for (int t = t0; t < t1; ++t, ++j) {
            wk.tile(m, ntp, prefix, KT);
            const int valid = wk.valid;
            const bool two = C::HALF < valid;
            if (wk.kvh != cur) cur = wk.kvh, ring_step(st, par, C::QB);  // the queries' slots: the softmax warps'
            if (is_v) ring_step(st, par, two ? 2 : 1);                   // the keys'
            const uint32_t s0 = st;
            as_wait(m, &m->r_full[st], par, ok);
            ring_step(st, par, 1);
            const uint32_t s1 = st;
            if (two) ring_step(st, par, 1);
            if (!is_v) ring_step(st, par, two ? 2 : 1);  // the values'
            const uint8_t *raw0 = sR + s0 * AS_SLOT, *raw1 = sR + s1 * AS_SLOT;
            const uint32_t own = cv::largest(raw0, raw1, w, lane, valid);
            if (lane == 0) m->cmax[is_v][j & 1][w] = own;
            if (is_v) asm volatile("bar.sync 6, %0;" ::"n"(AS_CONV * 32) : "memory");
            else asm volatile("bar.sync 5, %0;" ::"n"(AS_CONV * 32) : "memory");
            const uint32_t all = __reduce_max_sync(0xffffffffu, m->cmax[is_v][j & 1][lane & 3]);
            const int e = as_exponent(all);
            if (!is_v && j > 0) as_wait(m, &m->k_empty[0], (j - 1) & 1, ok);
            if (is_v && j > 1) as_wait(m, &m->v_empty[j & 1], ((j >> 1) - 1) & 1, ok);
            // behind these waits: P V of tile j - 2 followed the hand-over of O of tile j - 4,
            // whose scale stood in this word
            if (w == 0 && lane == 0) (is_v ? m->vsc : m->ksc)[j & 3] = as_pow2(e - 14);
            cv::store(raw0, raw1, is_v ? sV + (j & 1) * (C::NK * C::KPLANE) : sK, w, lane, valid, e);
            // (every value read has been stored: nothing of the slots is under way)
            if (lane == 0) {
                as_arrive(is_v ? &m->v_full[j & 1] : &m->k_full[0], ok);
                as_arrive(&m->r_empty[s0], ok);
                if (two) as_arrive(&m->r_empty[s1], ok);
            }
            wk.next(tpg);
        }
        }
    }
    } else {
        // ---------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFT_REGS));
        const int half = warp >> 2, q4 = warp & 3;
        const int row = q4 * 32 + lane, sq = row / G;
        const bool live = row < rows;
        const uint32_t lane_base = tmem + ((uint32_t)(q4 * 32) << 16);
        constexpr int HC = KT / 2, HD = DP / 2;  // this thread's keys of a tile, dims of the output
        constexpr float OFF = C::BF ? 0.f : C::ACC ? 6.f : 14.f;  // f16 weights: at most 2^14, small ones stay normal
        f2 o[HD / 2];
        float mrun = -INFINITY, lsum = 0.f, cprev = 1.f, qs = a.scale * AS_LOG2E;
        bool prev_act = false, prev_any = false;
        const uint32_t o_base = lane_base + C::O_COL + half * HD;

        // the row's f32 queries (this thread's half of the dims), scaled and split into TMEM
        auto load_q = [&](int seg) {  // seg: kv heads before this one in the run
            float4 v[HD / 4];
            float mx = 0.f;
            as_wait(m, &m->q_raw[seg & 1], (seg >> 1) & 1, ok);
            const uint8_t* src[HD / 32];
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) {
                const uint32_t blk = half * (HD / 32) + b;
                src[b] = sQ + blk * (AS_ROWS * 128);
                if (C::KF32) {  // a ring slot
                    uint32_t at = m->q_slot[seg & 1] + blk, par = m->q_par[seg & 1];
                    ring_step(at, par, 0);
                    as_wait(m, &m->r_full[at], par, ok);
                    src[b] = sR + at * AS_SLOT;
                }
            }
#pragma unroll
            for (int c = 0; c < HD / 4; ++c) {
                v[c] = *(const float4*)(src[c / 8] + row * 128 + ((c % 8 ^ (row & 7)) << 4));
                mx = as_max3(mx, fabsf(v[c].x), fabsf(v[c].y));
                mx = as_max3(mx, fabsf(v[c].z), fabsf(v[c].w));
            }
            m->mx[0][half][row] = mx;
            as_pair_sync(1 + q4);
            mx = fmaxf(mx, m->mx[0][half ^ 1][row]);
            const int e = as_exponent(__float_as_uint(mx));
            const float f = as_pow2(14 - e);
            qs = as_pow2(e - 14) * (a.scale * AS_LOG2E);
            const uint32_t dst = lane_base + C::Q_COL + half * (HD / 2);
#pragma unroll
            for (int c = 0; c < HD / 4; c += 4) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    as_split(v[c + i].x * f, v[c + i].y * f, hi[2 * i], lo[2 * i]);
                    as_split(v[c + i].z * f, v[c + i].w * f, hi[2 * i + 1], lo[2 * i + 1]);
                }
                as_st8(dst + 2 * c, hi);
                as_st8(dst + DP / 2 + 2 * c, lo);
            }
            as_wait_st();
            as_tc_before();
            __syncwarp();
            if (lane == 0) {
                as_arrive(&m->q_full, ok);
                as_arrive(&m->q_empty[seg & 1], ok);
            }
        };
        // ACC: the prefix's O (registers and buffer 0) times c
        auto rescale = [&](float c) {
            const f2 c2 = as_f2(c, c);
#pragma unroll
            for (int k = 0; k < HD / 2; ++k) o[k] = as_mul2(o[k], c2);
#pragma unroll 1
            for (int k = 0; k < HD; k += 32) {
                float x[32];
                as_ld32(o_base + k, x);
                as_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) as_un2(as_mul2(as_f2(x[i], x[i + 1]), c2), x[i], x[i + 1]);
#pragma unroll
                for (int i = 0; i < 32; i += 8) as_st8(o_base + k + i, reinterpret_cast<uint32_t*>(x) + i);
            }
            as_wait_st();
        };
        // ACC: the run's O joins the prefix's in registers
        auto bring = [&]() {
#pragma unroll
            for (int k = 0; k < HD; k += 32) {
                float x[32];
                as_ld32(o_base + k, x);
                as_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[k / 2 + i] = as_add2(o[k / 2 + i], as_f2(x[2 * i], x[2 * i + 1]));
            }
        };
        // scores of tile j -> weights of the rows that act, for the first h0 of this half's keys.
        // kq: the row's score factor (qs, times 2^exponent of an f32 tile); fix: an ACC prefix
        // tile behind the segment's first, whose O so far is rescaled when a maximum grows
        auto weigh = [&](int j, bool act, int h0, float kq, bool fix) {
            const uint32_t bf = j & 1, sb = lane_base + bf * C::S_COLS;
            float s[HC];
#pragma unroll
            for (int c = 0; c < HC; c += 32) as_ld32(sb + half * HC + c, s + c);
            as_wait_ld();
            if (h0 < HC || !act) {
                const int h = act ? h0 : 0;
#pragma unroll
                for (int k = 0; k < HC; ++k) s[k] = k < h ? s[k] : -INFINITY;
            }
            // (s stays unscaled; the scaled maximum is the maximum of the scaled, kq > 0)
            float m2[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < HC; k += 8)
#pragma unroll
                for (int q = 0; q < 4; ++q) m2[q] = as_max3(m2[q], s[k + 2 * q], s[k + 2 * q + 1]);
            const float mt = fmaxf(as_max3(m2[0], m2[1], m2[2]), m2[3]) * kq;
            m->mx[bf][half][row] = mt;
            as_pair_sync(1 + q4);  // (also: both halves of S are read, P may overwrite them)
            float cnew = 1.f;
            if (act) {
                // integer exponents: exact powers of two (0 on the first tile). ACC: the reference
                // only moves when it is passed by 2^8, as O in tensor memory then moves too
                const float top = ceilf(fmaxf(mt, m->mx[bf][half ^ 1][row]));
                const float mnew = top > mrun + (C::ACC ? 8.f : 0.f) ? top : mrun;
                if (mnew != mrun) cnew = as_ex2(mrun - mnew);  // (equal: also -inf, where no score was above it)
                lsum *= cnew;
                mrun = mnew;
            }
            if (C::ACC && fix && __any_sync(0xffffffffu, cnew != 1.f)) {
                as_wait(m, &m->o_full[bf ^ 1], ((j - 1) >> 1) & 1, ok);
                as_tc_after();
                rescale(cnew);
            }
            const float sub = act && mrun > -INFINITY ? OFF - mrun : 0.f;  // (no weight where -inf)
            const f2 q2 = as_f2(kq, kq), sub2 = as_f2(sub, sub);
            f2 l2[2] = {0ull, 0ull};
            // P over S: hi planes in the first half of the columns, lo in the second
#pragma unroll
            for (int k = 0; k < HC; k += 16) {
                uint32_t ph[8], pl[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float x, y;
                    as_un2(as_fma2(as_f2(s[k + 2 * i], s[k + 2 * i + 1]), q2, sub2), x, y);
                    x = as_ex2(x), y = as_ex2(y);
                    if (C::NP == 2) {
                        as_split(x, y, ph[i], pl[i]);
                    } else {
                        // the sum of the weights that V is multiplied by: where one of them dominates
                        // its rounding cancels
                        ph[i] = as_pack<C::BF>(x, y);
                        if (C::BF) {
                            x = __uint_as_float(ph[i] << 16), y = __uint_as_float(ph[i] & 0xffff0000u);
                        } else {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ph[i]));
                            x = f.x, y = f.y;
                        }
                    }
                    l2[i & 1] = as_add2(l2[i & 1], as_f2(x, y));
                }
                as_st8(sb + (half * HC + k) / 2, ph);
                if (C::NP == 2) as_st8(sb + KT / 2 + (half * HC + k) / 2, pl);
            }
            float x, y;
            as_un2(as_add2(l2[0], l2[1]), x, y);
            lsum += x + y;
            return cnew;
        };
        // the O of tile i, in buffer buf, joins the row's; or (ACC) stays, where i is of the prefix
        // and not its last tile before a suffix or the segment's end
        int taken = 0;  // ACC: hand-overs
        auto take_o = [&](int i, int buf, bool of_prefix) {
            as_wait(m, &m->o_full[i & 1], (i >> 1) & 1, ok);
            as_tc_after();
            if (C::ACC && of_prefix) {
                bring();
            } else if (prev_any) {
                // (an f32 tile's values come back to their scale here)
                const float vs = C::KF32 ? m->vsc[i & 3] : 1.f;
                const f2 c2 = as_f2(cprev, cprev), v2 = as_f2(vs, vs);
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    float x[32];
                    as_ld32(o_base + buf * DP + c, x);
                    as_wait_ld();
                    if (prev_act) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            f2& d = o[c / 2 + k];
                            const f2 xx = as_f2(x[2 * k], x[2 * k + 1]);
                            d = C::KF32 ? as_fma2(xx, v2, as_mul2(d, c2)) : as_fma2(d, c2, xx);
                        }
                    }
                }
            }
        };
        auto hand_over = [&](int b) {
            as_tc_before();
            __syncwarp();
            if (lane == 0) as_arrive(&m->o_empty[b], ok);
        };

        int j = 0, cur = -1, seg = -1, seg_t0 = t0;
        bool prev_pre = false;
        int nsuf = 0;  // ACC: suffix tiles of the segment so far
        AsWalk w;
        w.start(t0, tpg);
        for (int t = t0; t < t1; ++t, ++j) {
            const bool first = w.kvh != cur, of_prefix = w.off < ntp;
            w.tile(m, ntp, prefix, KT);
            if (first) {
                cur = w.kvh, seg_t0 = t;
                if constexpr (C::QF32) load_q(++seg);  // (the segment before is done with the last ones)
#pragma unroll
                for (int k = 0; k < HD / 2; ++k) o[k] = 0ull;
                nsuf = 0;
                mrun = -INFINITY;
                lsum = 0.f;
            }
            // the row's keys of this tile: all, or none
            const bool act = live && (of_prefix || sq == w.i);
            const bool any = __any_sync(0xffffffffu, act);
            const uint32_t bf = j & 1;
            as_wait(m, &m->s_full[bf], (j >> 1) & 1, ok);
            as_tc_after();
            float cnew = 1.f;
            if (any) {
                // (f32 queries: above 0, or the -inf of the keys that do not count would become NaN)
                const float kq = C::QF32 ? fmaxf(C::KF32 ? qs * m->ksc[j & 3] : qs, 1e-37f) : qs;
                cnew = weigh(j, act, w.valid - half * HC, kq, of_prefix && !first);
                // a new run starts: its first product waits for p_full, behind these reads
                if (C::ACC && of_prefix && !first && (t - seg_t0) % AS_RUN == 0) {
                    as_wait(m, &m->o_full[bf ^ 1], ((j - 1) >> 1) & 1, ok);
                    as_tc_after();
                    bring();
                }
            }
            as_wait_st();
            as_tc_before();
            __syncwarp();
            if (lane == 0) as_arrive(&m->p_full[bf], ok);
            if (C::ACC) {
                // (the first suffix tile of a segment without prefix tiles hands over all the same)
                if (!of_prefix) {
                    if (!first) take_o(j - 1, nsuf & 1, prev_pre);
                    hand_over(taken++ & 1);
                    ++nsuf;
                }
            } else if (!first) {
                take_o(j - 1, C::NOB == 2 ? (j - 1) & 1 : 0, false);
                hand_over(C::NOB == 2 ? (j - 1) & 1 : 0);
            }
            cprev = cnew, prev_act = act, prev_any = any, prev_pre = of_prefix;
            const bool end = t + 1 == t1 || w.off + 1 == tpg;
            w.next(tpg);
            if (!end) continue;

            // ---- the segment's last tile: add it, then the output or a partial
            take_o(j, C::ACC ? nsuf & 1 : C::NOB == 2 ? j & 1 : 0, C::ACC && prev_pre);
            if (C::ACC) {
                if (!prev_pre) hand_over(taken++ & 1);
            } else {
                hand_over(C::NOB == 2 ? j & 1 : 0);
            }
            m->lx[half][row] = lsum;
            as_pair_sync(1 + q4);
            float l = lsum + m->lx[half ^ 1][row];
            as_pair_sync(1 + q4);
            if (*(volatile int*)&m->fail) l = NAN;
            const int d0 = half * HD;
            const bool whole = seg_t0 == cur * tpg && t + 1 == (cur + 1) * tpg;
            const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
            const f2 inv2 = as_f2(inv, inv);
            // slot 1: a run that began in an earlier kv head; slot 0: the others
            const size_t ps = (size_t)blockIdx.x * 2 + (t0 < cur * tpg ? 1 : 0);
            const size_t at = (size_t)(seq0 + sq) * a.out_sn + (size_t)(cur * G + row % G) * a.out_sh + d0;
            if (!whole && live && half == 0) a.part_ml[ps * AS_ROWS + row] = make_float2(mrun, l);
            // (a row without keys here has no partial: mrun tells)
            const bool put = live && (whole || mrun != -INFINITY || isnan(l));
#pragma unroll
            for (int k = 0; k < HD; k += 8) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) as_un2(as_mul2(o[k / 2 + i], inv2), x[2 * i], x[2 * i + 1]);
                if (!put || d0 + k >= a.hd) continue;
                const bool two = d0 + k + 4 < a.hd;
                if (!whole) {
                    // [4 dims][128 rows]: neighbouring lanes write neighbouring addresses
                    float4* dst = a.part_o + (ps * 32 + (d0 + k) / 4) * AS_ROWS + row;
                    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                    if (two) dst[AS_ROWS] = make_float4(x[4], x[5], x[6], x[7]);
                } else if constexpr (C::QF32) {
                    float* dst = (float*)a.out + at + k;
                    *(float4*)dst = make_float4(x[0], x[1], x[2], x[3]);
                    if (two) *(float4*)(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
                } else {
                    *(uint4*)((uint16_t*)a.out + at + k) =
                        make_uint4(as_pack<C::BF>(x[0], x[1]), as_pack<C::BF>(x[2], x[3]), as_pack<C::BF>(x[4], x[5]),
                                   as_pack<C::BF>(x[6], x[7]));
                }
            }
        }
    }
    as_tc_before();
    __syncthreads();
    if (warp == C::WARPS - 1) {
        as_tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
    if (tid == 0 && a.error && *(volatile int*)&m->fail) atomicOr(a.error, 2u);
}

// Adds the partials of a (row tile, kv head) that several CTAs share, in CTA
// order: out = sum O_i 2^(m_i - m) / sum l_i 2^(m_i - m) (integer exponents). A
// warp takes 4 dims of 32 rows, a lane one row.
template <typename OT>
__global__ void __launch_bounds__(256) k_attn_merge(const __grid_constant__ AttnSharedArgs a) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int nd4 = (a.hd + 3) / 4;
    const int gw = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d4 = gw % nd4, rb = gw / nd4 % (AS_ROWS / 32), g = gw / nd4 / (AS_ROWS / 32);
    const int kvh = g % a.n_kv, rt = g / a.n_kv, row = rb * 32 + lane;
    const int n = a.n_dev ? *a.n_dev : a.n;
    const int G = a.group, spt = AS_ROWS / G, seq = rt * spt + row / G;
    if (rt * spt >= n || rb * 32 >= min(spt, n - rt * spt) * G) return;
    const int b0 = a.plan[3 * rt], nb = a.plan[3 * rt + 1], tpg = a.plan[3 * rt + 2];
    if (tpg == 0) return;
    const int total = tpg * a.n_kv;
    const int g0 = kvh * tpg, g1 = g0 + tpg;
    const int i0 = as_part_of(g0, total, nb), i1 = as_part_of(g1 - 1, total, nb);
    if (as_part(i0, total, nb) <= g0 && as_part(i0 + 1, total, nb) >= g1) return;  // written by its one CTA
    if (row >= spt * G || seq >= n) return;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // eight partials at a time, all their loads in flight (one that its CTA did not write is
    // read and not used)
    constexpr int MB = 8;
    const int q = total / nb, rem = total - q * nb;
    for (int i = i0; i <= i1; i += MB) {
        float2 x[MB];
        float4 v[MB];
#pragma unroll
        for (int k = 0; k < MB; ++k) {
            const int ii = min(i + k, i1), s0 = ii * q + min(ii, rem);
            const size_t ps = (size_t)(b0 + ii) * 2 + (s0 < g0 ? 1 : 0);
            x[k] = a.part_ml[ps * AS_ROWS + row];
            v[k] = a.part_o[(ps * 32 + d4) * AS_ROWS + row];
            if (i + k > i1 || (q == 0 && ii >= rem)) x[k] = make_float2(-INFINITY, 0.f);  // none, or a CTA without tiles
        }
        float mn = m;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < MB; ++k) mn = fmaxf(mn, x[k].x), bad |= isnan(x[k].y);
        const float c = mn == m ? 1.f : exp2f(m - mn);
        l *= c, o.x *= c, o.y *= c, o.z *= c, o.w *= c;
#pragma unroll
        for (int k = 0; k < MB; ++k) {
            const float cv = exp2f(x[k].x - mn);
            if (x[k].x == -INFINITY) continue;
            l = fmaf(x[k].y, cv, l);
            o.x = fmaf(v[k].x, cv, o.x), o.y = fmaf(v[k].y, cv, o.y);
            o.z = fmaf(v[k].z, cv, o.z), o.w = fmaf(v[k].w, cv, o.w);
        }
        if (bad) l = NAN;  // a CTA's wait ran out
        m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t at = (size_t)seq * a.out_sn + (size_t)(kvh * G + row % G) * a.out_sh + 4 * d4;
    if constexpr (sizeof(OT) == 4) {
        *(float4*)((float*)a.out + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
        constexpr bool BF = std::is_same<OT, __nv_bfloat16>::value;
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

// Workspace: [2 per CTA][128 rows] (m, l), the same rows' O, the row tiles' plan.
size_t attn_shared_work_bytes(int n, int group, int sms) {
    const size_t cta = as_grid(n, group, sms);
    return cta * 2 * AS_ROWS * (8 + 128 * 4) + (size_t)as_row_tiles(n, group) * 12 + 256;
}

typedef CUresult (*AsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static AsEncodeFn g_as_encode = nullptr;  // set by attn_shared_configure

// A map over [d3][d2][d1][d0] elements (strides in elements; a dimension of one
// element gets a stride that any map accepts) with boxes of [1][b2][b1][b0].
static cudaError_t as_map(CUtensorMap* out, CUtensorMapDataType type, int es, bool swizzle, const void* base, int rank,
                          const uint64_t* dim, const uint64_t* stride, const uint32_t* box) {
    cuuint64_t d[4], st[3];
    cuuint32_t b[4], one[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) d[i] = dim[i], b[i] = box[i];
    for (int i = 1; i < rank; ++i) st[i - 1] = dim[i] > 1 ? stride[i] * es : (dim[0] * es + 15) / 16 * 16;
    const CUresult r = g_as_encode(out, type, rank, const_cast<void*>(base), d, st, b, one,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int MODE, int DP>
static cudaError_t as_launch(AttnSharedArgs a, int sms, cudaStream_t s) {
    using C = AsCfg<MODE, DP>;
    const int R = as_row_tiles(a.n, a.group), spt = AS_ROWS / a.group;
    const CUtensorMapDataType type = C::KF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : C::BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    AsMaps maps{};
    const int es = C::KF32 ? 4 : 2;
    const uint32_t rows = C::KF32 ? C::HALF : C::KT, cols = C::KF32 ? DP : 64;
    cudaError_t e = cudaSuccess;
    {
        const uint64_t d[3] = {(uint64_t)a.hd, (uint64_t)a.n_kv * a.group, (uint64_t)a.n}, st[3] = {1, a.q_sh, a.q_sn};
        const uint32_t box[3] = {C::QF32 ? 32u : 64u, (uint32_t)a.group, (uint32_t)(spt < a.n ? spt : a.n)};
        e = as_map(&maps.q, C::QF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type, C::QF32 ? 4 : 2, true, a.q, 3, d, st, box);
    }
    if (e == cudaSuccess && a.prefix) {
        const uint64_t d[3] = {(uint64_t)a.hd, (uint64_t)a.n_kv, (uint64_t)a.prefix}, st[3] = {1, a.pre_sh, a.pre_st};
        const uint32_t box[3] = {cols, 1, rows};
        e = as_map(&maps.kp, type, es, !C::KF32, a.kp, 3, d, st, box);
        if (e == cudaSuccess) e = as_map(&maps.vp, type, es, !C::KF32, a.vp, 3, d, st, box);
    }
    if (e == cudaSuccess && a.slot_len) {
        const uint64_t d[4] = {(uint64_t)a.hd, (uint64_t)a.n_kv, (uint64_t)a.slot_len, (uint64_t)a.n_slots};
        const uint64_t st[4] = {1, a.slot_sh, a.slot_st, a.slot_ss};
        const uint32_t box[4] = {cols, 1, rows, 1};
        e = as_map(&maps.k, type, es, !C::KF32, a.k, 4, d, st, box);
        if (e == cudaSuccess) e = as_map(&maps.v, type, es, !C::KF32, a.v, 4, d, st, box);
    }
    if (e != cudaSuccess) return e;
    // Few tiles per (row tile, kv head): one CTA each, and no partials to add. Measured with
    // 4 sequences, 32 / 8 heads of 128 and 1, 2, 3, 4 tiles of a prefix, one CTA each against
    // all CTAs and the second kernel: bf16 9.3 / 10.3 / 12.3 / 14.4 us against 10.3 / 12.3 /
    // 12.3 / 12.3; f32 11.1 / 14.2 / 16.4 / 18.5 against 12.3 / 14.4 / 14.4 / 14.4. So it gains
    // up to two tiles and costs 2 to 4 us at the four it goes to.
    const long long most = (a.prefix + C::KT - 1) / C::KT +
                           (long long)(a.n < spt ? a.n : spt) * ((a.slot_len + C::KT - 1) / C::KT);
    a.whole = !a.prefix_dev && most <= 4 && (long long)R * a.n_kv <= 0x7fffffff;
    const int grid = a.whole ? R * a.n_kv : as_grid(a.n, a.group, sms);
    k_attn_shared<MODE, DP><<<grid, C::THREADS, C::SMEM, s>>>(a, maps);
    e = cudaGetLastError();
    if (e != cudaSuccess || a.whole) return e;
    cudaLaunchConfig_t cfg = {};
    const long long warps = (long long)R * a.n_kv * (AS_ROWS / 32) * ((a.hd + 3) / 4);
    cfg.gridDim = dim3((unsigned)((warps + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    using OT = typename std::conditional<MODE <= 1, float,
                                         typename std::conditional<MODE == 2, __half, __nv_bfloat16>::type>::type;
    return cudaLaunchKernelEx(&cfg, k_attn_merge<OT>, a);
}

cudaError_t launch_attn_shared(AttnSharedArgs a, int q_type, int kv_type, void* work, int sms, cudaStream_t s) {
    // the 16-bit caches' copies know neither rows that start behind the slot's first nor a
    // prefix that ends before its map does
    if ((a.slot_row0 || a.prefix_dev) && as_mode(q_type, kv_type) != 0) return cudaErrorInvalidValue;
    const size_t cta = as_grid(a.n, a.group, sms);
    a.part_ml = (float2*)work;
    a.part_o = (float4*)((uint8_t*)work + cta * 2 * AS_ROWS * 8);
    a.plan = (int*)((uint8_t*)work + cta * 2 * AS_ROWS * (8 + 128 * 4));
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
    if (!g_as_encode) {  // through the runtime's driver entry point (no link to libcuda)
        cudaDriverEntryPointQueryResult q;
        void* fn = nullptr;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess) return e;
        if (q != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
        g_as_encode = (AsEncodeFn)fn;
    }
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
