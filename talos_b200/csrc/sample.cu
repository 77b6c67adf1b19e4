// sample.cu -- the choice of a token from logits on B200 (sm_100a): temperature,
// top-k, top-p and min-p with one given random number per row (the truncations
// of Tsuskov/talos src/sample.rs:19-76, on the device).
//
// For a row of logits l with temperature T, in the order of descending logit
// (equal logits: the lower index first; NaN counts as -inf):
//   w_i = exp((l_i - max) / T), 0 for l_i = -inf
//   keep the first k; of these the shortest prefix with sum w >= p * (their sum);
//   of these the w_i >= m (the largest w is 1); W = sum of the kept w
//   the token is the first whose cumulative w exceeds u * W.
// All three truncations keep a prefix of the order, so each is known by its
// cumulative weight, and the choice is one search for a cumulative weight.
//
// Exactness. An answer is a border between cumulative sums, so weights are
// computed in f64 and summed as 64-bit integers in units of 2^-42: sums do not
// depend on their order, and a weight is off by at most 2^-42 (a million weights
// add up to less than 2^63). w = 2^-(k / 512) 2^(r / 512) with k the nearest integer
// to 512 log2(e) (max - l) / T: a table of 512 powers and the exponential's series to
// the third power (|r| <= 1/2: the fourth is below 9e-15), nine f64 operations where
// exp() took about a hundred instructions (64 rows of 128256: 117 -> 99 us).
//
// Bound: the weighing pass (about 50 instructions and two or three shared-memory atomics a
// logit for the exact weight), then the chain of phases, most of it in the leading CTA alone;
// over the kernel the issue slots are 42 % busy. 64 rows of 128256 f32: plain temperature
// 48 us (0.69 TB/s), top-p 62, top-k 35, mixed settings 58; 32 rows of 32000 with top-p 28
// us; one row of 32000 14-15 us.
//
// Structure: a cluster of 1 .. 8 CTAs takes a row; each CTA keeps its slice in
// shared memory, so the row is read from HBM once. No sort of the row: a
// histogram over 1024 bins of (max - l) / T (1/32 nat each or less; beyond 32 nats the
// weight is 0) counts and sums the weights per bin in shared memory, the CTAs add
// the cluster's histograms through distributed shared memory, the leading one scans
// the sum and finds the bins of the borders. When the elements up to the first
// truncating border are few (top-k, most top-p and min-p settings), they are
// gathered, ranked and finished in one step; otherwise each border's bin is
// gathered and ranked by itself. A bin that holds more elements than the list
// (equal or nearly equal logits) is split further by the bits of the
// (logit, index) key. The leading CTA drives; the others follow its commands.
#include <cooperative_groups.h>

#include "ops.cuh"

namespace cg = cooperative_groups;

namespace talos {

typedef unsigned long long u64;

constexpr int SP_THREADS = 512;
constexpr int SP_WARPS = SP_THREADS / 32;
constexpr int SP_NB = 1024;       // bins; two per thread
constexpr float SP_PER_NAT = 32;  // bins per nat
constexpr int SP_CAP = 1024;      // elements of a ranked list; two per thread
constexpr double SP_ONE = 4398046511104.0;  // 2^42
constexpr int SP_SLICE = 16384;  // logits of a row that one CTA keeps
constexpr int SP_IDX_BITS = 20;
static_assert(SP_THREADS == 512, "sp_pow's entries, one a thread");
static_assert((1 << SP_IDX_BITS) == SAMPLE_MAX_VOCAB, "index bits");

enum SpOp : int { SP_COUNT = 0, SP_WEIGH = 1, SP_GATHER_BINS = 2, SP_GATHER_KEYS = 3, SP_RANGE = 4, SP_SPLIT = 5,
                  SP_SUM_MIN = 6, SP_DONE = 7 };
struct SpCmd {
    int op, b0, b1, shift;
    u64 k0, k1;
};

struct SpSmem {
    uint32_t cnt[SP_NB], wlo[SP_NB], whi[SP_NB];
    u64 list[SP_CAP];  // leader: gathered keys, then the ranked ones
    u64 key[SP_CAP];   // this CTA's gathered keys; leader: keys by bucket
    u64 cum[SP_CAP];   // cumulative weights of the ranked list
    float cmax[8], cmin[8];  // each CTA's largest and smallest finite logit
    SpCmd cmd;
    uint32_t nlist;    // leader: gathered so far
    uint32_t mine, at; // gathered by this CTA, their place in the leader's list
    u64 ra, rb;        // this CTA's SP_RANGE (smallest, largest key) or SP_SUM_MIN (sum)
    u64 wa[SP_WARPS], wb[SP_WARPS];  // block scans
    float fa[SP_WARPS], fb[SP_WARPS];
    // result of a search
    uint32_t f_cnt, f_bin, f_at;
    u64 f_bc, f_bw;
    uint32_t keep;     // elements of the list with w >= min_p
    double pow[512];   // sp_pow
};

__device__ __forceinline__ float sp_load(float v) { return isnan(v) ? -INFINITY : v + 0.0f; }  // -0 -> +0
__device__ __forceinline__ float sp_load(__half v) { return sp_load(__half2float(v)); }
__device__ __forceinline__ float sp_load(__nv_bfloat16 v) { return sp_load(__bfloat162float(v)); }

// Position in the order: a smaller key comes first.
__device__ __forceinline__ u64 sp_key(float v, uint32_t i) { return ((u64)~total_order_key(v) << SP_IDX_BITS) | i; }
__device__ __forceinline__ float sp_key_value(u64 k) {
    const uint32_t o = ~(uint32_t)(k >> SP_IDX_BITS);
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

// 2^42 2^(-i / 512), i < 512: the product of 2^(-1 / 2) to 2^(-1 / 512) over i's bits.
__device__ __forceinline__ double sp_pow(int i) {
    constexpr double root[9] = {0.99864711289097017, 0.99729605608547012, 0.99459942348363317,
                                0.98922801319397548, 0.97857206208770013, 0.95760328069857365,
                                0.91700404320467123, 0.84089641525371454, 0.70710678118654752};
    double w = SP_ONE;
#pragma unroll
    for (int b = 0; b < 9; ++b)
        if (i >> b & 1) w *= root[b];
    return w;
}

struct SpScale {
    double vmax, c;  // c: 512 log2(e) / T
};
// f32 -> f64 by its bits (two integer operations where the conversion runs at a quarter
// of their rate). Zeros and denormals become 2^-126 to 2^-125, which matters below a
// temperature of 1e-24 only.
__device__ __forceinline__ double sp_f64(float v) {
    const uint32_t b = __float_as_uint(v), m = b & 0x7fffffffu;
    return __hiloint2double((int)((b & 0x80000000u) | ((m >> 3) + (896u << 20))), (int)(m << 29));
}
// 2^42 w of a value v whose bin is below SP_NB, plus `base` (a power of two, or 0). At the
// maximum, +inf included, the difference is 0 and w is 2^42 exactly.
__device__ __forceinline__ double sp_weight(float v, const SpScale& q, const double* pow, double base) {
    const double t = (q.vmax - sp_f64(v)) * q.c;
    const double round = 6755399441055744.0;  // 1.5 2^52: the sum's low word is the nearest integer
    const double tm = t + round;
    const int k = __double2loint(tm);
    const double r = (tm - round) - t;
    constexpr double h = 0.0013538030870311431;  // ln 2 / 512
    const double e = fma(r, fma(r, fma(r, h * h * h / 6, h * h / 2), h), 1.0);
    const double p = pow[k & 511];
    return fma(__hiloint2double(__double2hiint(p) - ((k >> 9) << 20), __double2loint(p)), e, base);  // 2^-(k / 512)
}
// To the nearest integer (w <= 2^42).
__device__ __forceinline__ u64 sp_fixed(float v, const SpScale& q, const double* pow) {
    return (u64)__double_as_longlong(sp_weight(v, q, pow, 4503599627370496.0)) & 0xfffffffffffffull;  // 2^52
}
// The bins: bin of v = half (vmax - v) scale. half is 1/2 where vmax - v can pass the largest
// f32 (the product with it is exact in the fma), else 1.
struct SpBins {
    float vmax, top, half, scale;  // top: half vmax
};
// Bin of value v, SP_NB for weight 0. Non-decreasing as v falls: every rounding here is monotone.
__device__ __forceinline__ float sp_z(float v, const SpBins& g) {
    return v == g.vmax ? 0.f : __fmul_rn(__fmaf_rn(-g.half, v, g.top), g.scale);
}
__device__ __forceinline__ int sp_bin(float v, const SpBins& g) {
    const float z = sp_z(v, g);
    return z < (float)SP_NB ? (int)z : SP_NB;  // NaN (-inf at a scale of 0) gives SP_NB
}

// Exclusive block scan of (a, b); returns the totals through ta, tb.
__device__ __forceinline__ void sp_scan(SpSmem& s, u64& a, u64& b, u64& ta, u64& tb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 x = a, y = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) x += p, y += q;
    }
    __syncthreads();
    if (lane == 31) s.wa[warp] = x, s.wb[warp] = y;
    __syncthreads();
    u64 px = 0, py = 0;
    ta = tb = 0;
#pragma unroll
    for (int w = 0; w < SP_WARPS; ++w) {
        if (w == warp) px = ta, py = tb;
        ta += s.wa[w], tb += s.wb[w];
    }
    a = px + x - a;
    b = py + y - b;
}

// RES: the CTA's slice of the row stays in shared memory (up to SP_SLICE
// logits as f32); otherwise every pass reads it again (vocabularies above
// 8 x SP_SLICE, or fewer CTAs a row). (In registers, 32 logits a thread, the f64 weights spilled.)
template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(SP_THREADS, 2) k_sample(const __grid_constant__ SampleArgs a, int slice) {
    __shared__ SpSmem s;
    extern __shared__ __align__(16) float vals[];  // RES: [slice]
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C;
    if (a.n_dev && row >= *a.n_dev) return;  // (the whole cluster)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int VW = 16 / (int)sizeof(T);
    SpSmem* lead = cluster.map_shared_rank(&s, 0);
    const int i0 = min(a.vocab, rank * slice), n_own = min(a.vocab, i0 + slice) - i0;
    const T* lg = (const T*)a.logits + (size_t)row * a.stride + i0;

    float mx = -INFINITY, mn = INFINITY;
    auto minmax = [&](float v) {
        mx = fmaxf(mx, v);
        mn = fminf(mn, v > -INFINITY ? v : INFINITY);
    };
    if (VEC) {  // slice is a multiple of VW, so lg is 16-byte aligned
#pragma unroll 4
        for (int i = tid * VW; i < n_own; i += SP_THREADS * VW) {
            float v[VW];
            if (i + VW <= n_own) {
                const uint4 q = ldg_stream_u4(lg + i);
                const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
                for (int k = 0; k < VW; ++k) v[k] = sp_load(t[k]);
            } else {
#pragma unroll
                for (int k = 0; k < VW; ++k) v[k] = i + k < n_own ? sp_load(lg[i + k]) : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < VW; ++k) minmax(v[k]);
#pragma unroll
            for (int k = 0; k < VW; k += 4)
                if (RES) *(float4*)(vals + i + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
        }
    } else {
#pragma unroll 8
        for (int i = tid; i < n_own; i += SP_THREADS) {
            const float v = sp_load(lg[i]);
            if (RES) vals[i] = v;
            minmax(v);
        }
    }
    // the slice's last four start on a multiple of four (-inf has weight 0)
    if (RES && tid < 4 && n_own + tid < (n_own + 3) / 4 * 4) vals[n_own + tid] = -INFINITY;
    auto each = [&](auto&& f) {  // (after the barriers of the maximum)
        if (RES) {
#pragma unroll 2
            for (int i = 4 * tid; i < n_own; i += 4 * SP_THREADS) {
                const float4 v = *(const float4*)(vals + i);
                f(v.x, (uint32_t)(i0 + i));
                f(v.y, (uint32_t)(i0 + i + 1));
                f(v.z, (uint32_t)(i0 + i + 2));
                f(v.w, (uint32_t)(i0 + i + 3));
            }
        } else if (VEC) {
            const int nv = n_own / VW * VW;
#pragma unroll 2
            for (int i = tid * VW; i < nv; i += SP_THREADS * VW) {
                const uint4 x = __ldg((const uint4*)(lg + i));
                const T* t = reinterpret_cast<const T*>(&x);
#pragma unroll
                for (int k = 0; k < VW; ++k) f(sp_load(t[k]), (uint32_t)(i0 + i + k));
            }
            if (tid < n_own - nv) f(sp_load(lg[nv + tid]), (uint32_t)(i0 + nv + tid));
        } else {
#pragma unroll 4
            for (int i = tid; i < n_own; i += SP_THREADS) f(sp_load(lg[i]), (uint32_t)(i0 + i));
        }
    };

    // settings of the row; T <= 0 (or NaN) is the greedy choice: the first of the order
    float temp = a.temperature_dev ? a.temperature_dev[row] : a.temperature;
    int topk = a.top_k_dev ? a.top_k_dev[row] : a.top_k;
    const float topp = a.top_p_dev ? a.top_p_dev[row] : a.top_p;
    float minp = a.min_p_dev ? a.min_p_dev[row] : a.min_p;
    minp = minp > 0.f ? fminf(minp, 1.0f) : 0.f;  // NaN: off
    if (!(temp > 0.f)) temp = 1.f, topk = 1;
    const double inv_t = fmin(1.0 / (double)temp, 1e30);
    s.pow[tid] = sp_pow(tid);

    // the row's largest and smallest finite logit
    mx = warp_max(mx);
    mn = -warp_max(-mn);
    if (lane == 0) s.fa[warp] = mx, s.fb[warp] = mn;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < SP_WARPS ? s.fa[lane] : -INFINITY);
        mn = -warp_max(lane < SP_WARPS ? -s.fb[lane] : -INFINITY);
        if (lane < C) {
            SpSmem* o = cluster.map_shared_rank(&s, lane);
            o->cmax[rank] = mx, o->cmin[rank] = mn;
        }
    }
    cluster.sync();
    float vmax = s.cmax[0], vmin = s.cmin[0];
    for (int c = 1; c < C; ++c) vmax = fmaxf(vmax, s.cmax[c]), vmin = fminf(vmin, s.cmin[c]);
    if (vmax == -INFINITY) {  // nothing to choose from; the whole cluster agrees
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.f;
        }
        return;
    }

    const SpScale q{sp_f64(vmax), inv_t * 738.65986093514925};  // 512 log2(e)
    // Bins per logit: the row's range over all bins, at most 32 nats (the smallest logit's
    // bin is below SP_NB for every rounding; an infinite or empty range leaves the 32 nats).
    // With 32 nats always, rows of 128256 with a deviation of 1.5 nats had bins of more than
    // SP_CAP and took 193,000 clocks instead of 85,000 (64 rows with top-p: 105 -> 63 us).
    // (1e30: logits closer than 1e-27 to each other all lie in bin 0, where an infinite
    // scale would leave the maximum alone.)
    const float half = vmax < INFINITY && !(vmax - vmin < INFINITY) ? 0.5f : 1.f;
    const float per_nat = SP_PER_NAT / half;
    const SpBins bins{vmax, half * vmax, half,
                      fmaxf((float)inv_t * per_nat,
                            fminf((float)(SP_NB - 1) / fmaf(-half, vmin, half * vmax), 1e30f))};
    const double min_w = (double)minp * SP_ONE;

    auto zero_hist = [&]() {
        for (int b = tid; b < SP_NB; b += SP_THREADS) s.cnt[b] = 0, s.wlo[b] = 0, s.whi[b] = 0;
        __syncthreads();
    };
    auto add_hist = [&](int b, u64 w) {
        // 64-bit add as two 32-bit ones: the carry comes from the value that the low word had
        const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.wlo[b], lo);
        const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&s.whi[b], hi);
    };
    // matches are collected here and handed to the leader at once (one atomic on the
    // leader's counter for each took 8,000 clocks for 600 keys, this 3,000)
    auto gather = [&](u64 k) {
        const uint32_t at = atomicAdd(&s.mine, 1u);
        if (at < SP_CAP) s.key[at] = k;
    };
    auto hand_over = [&]() {
        __syncthreads();
        const uint32_t n = s.mine;
        if (tid == 0 && n) s.at = atomicAdd(&lead->nlist, n);
        __syncthreads();
        if (tid == 0) s.mine = 0;
        for (uint32_t i = tid; i < n && i < SP_CAP && s.at + i < SP_CAP; i += SP_THREADS)
            lead->list[s.at + i] = s.key[i];
    };
    // Each CTA adds its share of the bins over the cluster and hands the sums to the
    // leader, in place of its list and cum (the leader alone, reading 8 x 12 KB, took
    // 4,500 clocks; this and its barrier 4,000, beside the others' work).
    auto sum_hist = [&]() {
        cluster.sync();
        const int nb = SP_NB / C;  // C is a power of two
        for (int b = rank * nb + tid; b < (rank + 1) * nb; b += SP_THREADS) {
            uint32_t n = 0;
            u64 w = 0;
#pragma unroll 8
            for (int c = 0; c < C; ++c) {
                const SpSmem* o = cluster.map_shared_rank(&s, c);
                n += o->cnt[b];
                w += ((u64)o->whi[b] << 32) + o->wlo[b];
            }
            ((uint32_t*)lead->cum)[b] = n;
            lead->list[b] = w;
        }
    };
    // one command, by every CTA of the cluster
    auto execute = [&](const SpCmd& c) {
        switch (c.op) {
            case SP_COUNT:
            case SP_WEIGH:
                zero_hist();
                each([&](float v, uint32_t) {
                    const int b = sp_bin(v, bins);
                    if (b < SP_NB) {
                        atomicAdd(&s.cnt[b], 1u);
                        if (c.op == SP_WEIGH) add_hist(b, sp_fixed(v, q, s.pow));
                    }
                });
                sum_hist();
                break;
            case SP_GATHER_BINS: {
                const float z0 = (float)c.b0, z1 = (float)(c.b1 + 1);  // b0 <= bin <= b1
                each([&](float v, uint32_t i) {
                    const float z = sp_z(v, bins);
                    if (z >= z0 && z < z1) gather(sp_key(v, i));
                });
                hand_over();
                break;
            }
            case SP_GATHER_KEYS:
                each([&](float v, uint32_t i) {
                    const u64 k = sp_key(v, i);
                    if (k >= c.k0 && k <= c.k1 && sp_bin(v, bins) < SP_NB) gather(k);
                });
                hand_over();
                break;
            case SP_RANGE: {
                u64 lo = ~0ull, hi = 0ull;
                each([&](float v, uint32_t i) {
                    if (sp_bin(v, bins) == c.b0) {
                        const u64 k = sp_key(v, i);
                        lo = k < lo ? k : lo;
                        hi = k > hi ? k : hi;
                    }
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const u64 p = __shfl_xor_sync(0xffffffffu, lo, o), q = __shfl_xor_sync(0xffffffffu, hi, o);
                    lo = p < lo ? p : lo;
                    hi = q > hi ? q : hi;
                }
                // (64-bit atomics in another CTA's shared memory lost updates: each CTA
                // leaves its own result for the leader to read)
                if (lane == 0) s.wa[warp] = lo, s.wb[warp] = hi;
                __syncthreads();
                if (tid == 0) {
                    for (int w = 1; w < SP_WARPS; ++w) {
                        lo = s.wa[w] < lo ? s.wa[w] : lo;
                        hi = s.wb[w] > hi ? s.wb[w] : hi;
                    }
                    s.ra = lo, s.rb = hi;
                }
                break;
            }
            case SP_SPLIT:
                zero_hist();
                each([&](float v, uint32_t i) {
                    const u64 k = sp_key(v, i);
                    if (k >= c.k0 && k <= c.k1 && sp_bin(v, bins) < SP_NB) {
                        const int b = (int)((k - c.k0) >> c.shift);
                        atomicAdd(&s.cnt[b], 1u);
                        add_hist(b, sp_fixed(v, q, s.pow));
                    }
                });
                sum_hist();
                break;
            case SP_SUM_MIN: {
                u64 sum = 0;
                each([&](float v, uint32_t) {
                    if (sp_bin(v, bins) < SP_NB) {
                        if (sp_weight(v, q, s.pow, 0.0) >= min_w) sum += sp_fixed(v, q, s.pow);
                    }
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0) s.wa[warp] = sum;
                __syncthreads();
                if (tid == 0) {
                    for (int w = 1; w < SP_WARPS; ++w) sum += s.wa[w];
                    s.ra = sum;
                }
                break;
            }
        }
    };

    // with a top-k that fits the list, counts alone find the candidates; the
    // weights of all elements are only needed without one
    const bool count_only = topk > 0 && topk <= SP_CAP / 2;
    const SpCmd first{count_only ? SP_COUNT : SP_WEIGH, 0, 0, 0, 0, 0};
    if (tid == 0) s.nlist = s.mine = 0;
    execute(first);
    cluster.sync();
    if (rank != 0) {
        for (;;) {
            cluster.sync();  // the leader has written this CTA's cmd
            const SpCmd c = s.cmd;
            if (c.op == SP_DONE) return;
            execute(c);
            cluster.sync();
        }
    }

    // ---------------------------------------------------------- the leading CTA
    auto step = [&](const SpCmd& c) {
        __syncthreads();
        if (tid < C) cluster.map_shared_rank(&s, tid)->cmd = c;
        if (tid == 0) s.nlist = 0;
        cluster.sync();
        execute(c);
        cluster.sync();
    };
    // the cluster's histogram: this thread's two bins and what lies before them
    uint32_t c0, c1;
    u64 w0, w1, bc, bw, tc, tw;
    auto load_hist = [&]() {
        const uint2 n = *(const uint2*)((const uint32_t*)s.cum + 2 * tid);
        c0 = n.x, c1 = n.y;
        w0 = s.list[2 * tid], w1 = s.list[2 * tid + 1];
        bc = (u64)c0 + c1, bw = w0 + w1;
        sp_scan(s, bc, bw, tc, tw);
    };
    // first bin whose cumulative count (or weight), on top of (xc, xw), reaches x >= 1
    auto find = [&](bool by_count, u64 x, u64 xc, u64 xw) {
        __syncthreads();
        if (tid == 0) s.f_bin = 0, s.f_cnt = 0, s.f_bc = xc, s.f_bw = xw;
        __syncthreads();
        const u64 b = by_count ? xc + bc : xw + bw, p = by_count ? (u64)c0 : w0, q = by_count ? (u64)c1 : w1;
        if (b < x && x <= b + p) s.f_bin = 2 * tid, s.f_cnt = c0, s.f_bc = xc + bc, s.f_bw = xw + bw;
        if (b + p < x && x <= b + p + q)
            s.f_bin = 2 * tid + 1, s.f_cnt = c1, s.f_bc = xc + bc + c0, s.f_bw = xw + bw + w0;
        __syncthreads();
    };
    // sort the gathered list (keys are unique) and sum its weights. The keys are put into
    // 1024 buckets by their leading bits and each counts the smaller ones of its own bucket
    // (600 keys: 2,500 clocks; counting over the whole list or a sorting network: 15,000)
    u64 lx = 0, l0 = 0, l1 = 0;  // this thread's two: weights, and the sum before them
    auto rank_list = [&](int n) {
        u64 k[2], lo = ~0ull, hi = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = tid + j * SP_THREADS;
            k[j] = i < n ? s.list[i] : 0;
            if (i < n) lo = k[j] < lo ? k[j] : lo, hi = k[j] > hi ? k[j] : hi;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const u64 x = __shfl_xor_sync(0xffffffffu, lo, o), y = __shfl_xor_sync(0xffffffffu, hi, o);
            lo = x < lo ? x : lo;
            hi = y > hi ? y : hi;
        }
        __syncthreads();
        if (lane == 0) s.wa[warp] = lo, s.wb[warp] = hi;
        *(uint2*)&s.cnt[2 * tid] = make_uint2(0, 0);
        if (tid == 0) s.keep = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SP_WARPS; ++w) {
            lo = s.wa[w] < lo ? s.wa[w] : lo;
            hi = s.wb[w] > hi ? s.wb[w] : hi;
        }
        const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
        uint32_t at[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (tid + j * SP_THREADS < n) at[j] = atomicAdd(&s.cnt[(k[j] - lo) >> shift], 1u);
        __syncthreads();
        const uint2 c = *(const uint2*)&s.cnt[2 * tid];
        u64 ex = c.x + c.y, dummy = 0, t1, t2;
        sp_scan(s, ex, dummy, t1, t2);
        *(uint2*)&s.wlo[2 * tid] = make_uint2((uint32_t)ex, (uint32_t)ex + c.x);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (tid + j * SP_THREADS < n) s.key[s.wlo[(k[j] - lo) >> shift] + at[j]] = k[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (tid + j * SP_THREADS < n) {
                const uint32_t b = (uint32_t)((k[j] - lo) >> shift), b0 = s.wlo[b], nb = s.cnt[b];
                uint32_t pos = b0;
                for (uint32_t i = 0; i < nb; ++i) pos += s.key[b0 + i] < k[j] ? 1 : 0;
                s.list[pos] = k[j];
            }
        __syncthreads();
        u64 x[2] = {0, 0};
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            if (i < n) {
                const float v = sp_key_value(s.list[i]);
                x[j] = sp_fixed(v, q, s.pow);
                keep += sp_weight(v, q, s.pow, 0.0) >= min_w ? 1u : 0u;
            }
        }
        l0 = x[0], l1 = x[1];
        lx = l0 + l1, dummy = 0;
        sp_scan(s, lx, dummy, t1, t2);
        if (2 * tid < n) s.cum[2 * tid] = lx + l0;
        if (2 * tid + 1 < n) s.cum[2 * tid + 1] = lx + l0 + l1;
        if (keep) atomicAdd(&s.keep, keep);
        __syncthreads();
    };
    // first of the ranked list with base + cum >= x, else its last (all threads get it)
    auto list_find = [&](int n, u64 base, u64 x) {
        if (tid == 0) s.f_at = n - 1;
        __syncthreads();
        if (base + lx < x && x <= base + lx + l0) s.f_at = 2 * tid;
        if (base + lx + l0 < x && x <= base + lx + l0 + l1) s.f_at = 2 * tid + 1;
        __syncthreads();
        const int j = (int)s.f_at;
        __syncthreads();
        return j;
    };
    auto p_target = [&](u64 z) {  // smallest integer >= p * z, within 1 .. z
        const double t = ceil((double)topp * (double)z);
        return t < 1.0 ? 1ull : (t >= (double)z ? z : (u64)t);
    };
    auto draw_target = [&](u64 w) {  // first cumulative weight > u * W
        const double t = floor((double)a.u[row] * (double)w);
        const u64 x = t > 0.0 ? (t >= (double)w ? w - 1 : (u64)t) : 0ull;  // NaN: 0
        return (x >= w ? w - 1 : x) + 1;
    };
    u64 chosen = 0, W = 0;
    load_hist();
    // the last bin that any truncation can keep
    int bcut = SP_NB;
    u64 ncut = tc;
    const bool k_active = topk > 0 && (u64)topk < tc;
    if (k_active) {
        find(true, (u64)topk, 0, 0);
        bcut = (int)s.f_bin, ncut = s.f_bc + s.f_cnt;
    }
    // (top-p is a share of the top-k's weight: with both, the list holds the whole top-k)
    const bool sum_known = !k_active && !count_only;
    if (minp > 0.f && (sum_known || !(topp < 1.f))) {
        // w < m beyond -ln m nats; one bin more covers the roundings of both
        const float zb = -logf(minp) * (half * bins.scale / (float)inv_t) + 2.0f;
        const int b = zb < (float)(SP_NB - 1) ? (int)zb : SP_NB - 1;
        if (b < bcut) {
            __syncthreads();
            if (tid == b / 2) s.f_bc = bc + c0 + (b & 1 ? c1 : 0);
            __syncthreads();
            if (s.f_bc < ncut) ncut = s.f_bc;
            bcut = b;
        }
    }
    if (topp < 1.f && sum_known) {
        find(false, p_target(tw), 0, 0);
        if ((int)s.f_bin < bcut) bcut = (int)s.f_bin, ncut = s.f_bc + s.f_cnt;
    }
    if (ncut <= SP_CAP) {
        // everything that can be kept fits the list
        const int n = (int)ncut;
        step(SpCmd{SP_GATHER_BINS, 0, bcut < SP_NB ? bcut : SP_NB - 1, 0, 0, 0});
        rank_list(n);
        int keep = n;
        u64 z = tw;  // weight under top-k
        if (!sum_known) {
            if (topk < keep) keep = topk;
            z = s.cum[keep - 1];
        }
        if (topp < 1.f) {
            const int j = list_find(n, 0, p_target(z)) + 1;
            if (j < keep) keep = j;
        }
        if (minp > 0.f && (int)s.keep < keep) keep = (int)s.keep;
        if (keep < 1) keep = 1;
        W = s.cum[keep - 1];
        const int j = list_find(n, 0, draw_target(W));
        chosen = s.list[j];
    } else {
        if (count_only) {  // more equal logits at the border than the list holds
            step(SpCmd{SP_WEIGH, 0, 0, 0, 0, 0});
            load_hist();
        }
        const uint32_t hc0 = c0, hc1 = c1;
        const u64 hw0 = w0, hw1 = w1, hbc = bc, hbw = bw, htw = tw;
        // the element at cumulative count / weight x: its bin, then its place in
        // the bin. Returns the cumulative weight up to and with it.
        auto resolve = [&](bool by_count, u64 x) {
            c0 = hc0, c1 = hc1, w0 = hw0, w1 = hw1, bc = hbc, bw = hbw;
            find(by_count, x, 0, 0);
            uint32_t n = s.f_cnt;
            u64 xc = s.f_bc, xw = s.f_bw;
            const int b = (int)s.f_bin;
            if (n <= SP_CAP) {
                step(SpCmd{SP_GATHER_BINS, b, b, 0, 0, 0});
            } else {
                step(SpCmd{SP_RANGE, b, b, 0, 0, 0});
                u64 k0 = ~0ull, k1 = 0;
                for (int q = 0; q < C; ++q) {
                    const SpSmem* o = cluster.map_shared_rank(&s, q);
                    k0 = o->ra < k0 ? o->ra : k0;
                    k1 = o->rb > k1 ? o->rb : k1;
                }
                while (n > SP_CAP) {
                    int shift = 0;
                    while (((k1 - k0) >> shift) >= SP_NB) ++shift;
                    step(SpCmd{SP_SPLIT, 0, 0, shift, k0, k1});
                    load_hist();
                    find(by_count, x, xc, xw);
                    n = s.f_cnt, xc = s.f_bc, xw = s.f_bw;
                    k0 += (u64)s.f_bin << shift;
                    const u64 last = k0 + ((1ull << shift) - 1);
                    k1 = last < k1 ? last : k1;
                }
                step(SpCmd{SP_GATHER_KEYS, 0, 0, 0, k0, k1});
            }
            rank_list((int)n);
            const int j = by_count ? (int)(x - xc) - 1 : list_find((int)n, xw, x);
            chosen = s.list[j];
            const u64 cum = xw + s.cum[j];
            __syncthreads();
            return cum;
        };
        W = htw;
        if (k_active) W = resolve(true, (u64)topk);
        if (topp < 1.f) W = resolve(false, p_target(W));
        if (minp > 0.f) {
            step(SpCmd{SP_SUM_MIN, 0, 0, 0, 0, 0});
            u64 sum = 0;
            for (int q = 0; q < C; ++q) sum += cluster.map_shared_rank(&s, q)->ra;
            if (sum < W) W = sum;
        }
        resolve(false, draw_target(W));
    }
    if (tid == 0) {
        a.tokens[row] = (int32_t)(chosen & (SAMPLE_MAX_VOCAB - 1));
        if (a.probs)
            a.probs[row] = (float)(sp_weight(sp_key_value(chosen), q, s.pow, 0.0) / (double)W);
    }
    __syncthreads();
    if (tid < C) cluster.map_shared_rank(&s, tid)->cmd.op = SP_DONE;
    cluster.sync();
}

template <typename T, bool RES, bool VEC>
static cudaError_t launch_one(const SampleArgs& a, int C, int slice, cudaStream_t s) {
    auto* k = k_sample<T, RES, VEC>;
    const size_t smem = RES ? (size_t)slice * 4 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.n * C);
    cfg.blockDim = dim3(SP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, a, slice);
}

template <typename T>
static cudaError_t launch_type(const SampleArgs& a, int sms, cudaStream_t s) {
    // CTAs per row: enough that a slice fits, then more (down to 4096 logits
    // each) while all of them still run at once, two per SM
    int C = 1;
    while (C < 8 && (long)C * SP_SLICE < a.vocab) C *= 2;
    while (C < 8 && (long)C * 4096 < a.vocab && 2L * C * a.n <= 2L * sms) C *= 2;
    // Rows that would not all run at once take half as many CTAs where those do, which read
    // their slices again from L2 where they no longer fit (64 rows of 128256, plain
    // temperature: 8 CTAs a row in two waves 60 us, 4 in one 50).
    if (C > 1 && (long)C * a.n > 2L * sms && (long)C / 2 * a.n <= 2L * sms) C /= 2;
    const int slice = ((a.vocab + C - 1) / C + 15) / 16 * 16;
    const bool res = slice <= SP_SLICE;
    const bool vec = ((uintptr_t)a.logits % 16 == 0) && (a.stride * sizeof(T)) % 16 == 0;
    return res ? vec ? launch_one<T, true, true>(a, C, slice, s) : launch_one<T, true, false>(a, C, slice, s)
               : vec ? launch_one<T, false, true>(a, C, slice, s) : launch_one<T, false, false>(a, C, slice, s);
}

// Opt-in shared memory of the current device's kernels (once per device).
cudaError_t sample_configure() {
    auto set = [](const void* k) {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SP_SLICE * 4);
    };
    const void* ks[] = {(const void*)k_sample<float, true, true>,         (const void*)k_sample<float, true, false>,
                        (const void*)k_sample<__half, true, true>,        (const void*)k_sample<__half, true, false>,
                        (const void*)k_sample<__nv_bfloat16, true, true>, (const void*)k_sample<__nv_bfloat16, true, false>};
    for (const void* k : ks) {
        const cudaError_t e = set(k);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_sample(const SampleArgs& a, int type, int sms, cudaStream_t s) {
    switch (type) {
        case DT_F32: return launch_type<float>(a, sms, s);
        case DT_F16: return launch_type<__half>(a, sms, s);
        case DT_BF16: return launch_type<__nv_bfloat16>(a, sms, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace talos
