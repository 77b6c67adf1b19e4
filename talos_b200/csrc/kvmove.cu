// kvmove.cu -- rows moved between cache slots on B200 (sm_100a): a prompt
// copied (forked) into other slots, live slots compacted to the front.
//
// A move copies rows [start, start + len) of slot src to slot dst, in every
// array (K, V) and layer. The moves of a call are simultaneous: every read sees
// the data from before the call. The host orders them so that each slot is read
// by all its readers before it is overwritten, and groups them into components
// that touch disjoint slots; a cycle of slots keeps one chunk aside (MOVE_TMP).
// A thread takes one offset of a component (array, layer, row, 16 bytes of the
// row) and carries out all of the component's moves at that offset, so the
// order between them is its own program order: no barrier, no second buffer,
// and a slot copied to many others is read once.
//
// Bound: HBM. Each source row is read once, each destination row written once.
#include <string.h>

#include "ops.cuh"

namespace talos {

constexpr int MV_THREADS = 256;

template <int CAP>
struct MoveProg {
    MoveGeom g;
    int n_comp;
    uint32_t comp[CAP + 1];    // first instruction of each component
    uint32_t block[CAP + 1];   // first block of each component
    uint32_t row0[CAP];        // rows the component touches: row0 ..
    uint32_t rows[CAP];        //   row0 + rows - 1
    MoveIns ins[CAP + CAP / 2];  // a cycle (two moves at least) adds one instruction
};

template <int VEC>
struct MvWord;
template <>
struct MvWord<16> {
    using T = uint4;
};
template <>
struct MvWord<8> {
    using T = uint2;
};
template <>
struct MvWord<4> {
    using T = uint32_t;
};
template <>
struct MvWord<2> {
    using T = uint16_t;
};
template <>
struct MvWord<1> {
    using T = uint8_t;
};

// OFF offsets per thread, BAT instructions whose loads are in flight together:
// loads may run ahead of earlier stores because no slot is read after it was written.
constexpr int MV_OFF = 4, MV_BAT = 4;

template <int VEC, int CAP>
__global__ void __launch_bounds__(MV_THREADS) k_kv_move(const __grid_constant__ MoveProg<CAP> p) {
    using T = typename MvWord<VEC>::T;
    int lo = 0, hi = p.n_comp;  // the component of this block
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.block[mid] <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const uint32_t cpr = (uint32_t)(p.g.row_bytes / VEC);  // chunks per row
    const unsigned long long span = (unsigned long long)p.rows[lo] * cpr;
    const uint32_t per_outer = (uint32_t)((span + MV_THREADS * MV_OFF - 1) / (MV_THREADS * MV_OFF));
    const uint32_t b = blockIdx.x - p.block[lo];
    const uint32_t outer = b / per_outer;  // (array, layer)
    uint8_t* base = p.g.base[outer / p.g.n_outer] + (size_t)(outer % p.g.n_outer) * p.g.outer_stride;
    const unsigned long long i0 = (unsigned long long)(b % per_outer) * (MV_THREADS * MV_OFF) + threadIdx.x;
    uint32_t row[MV_OFF];
    size_t off[MV_OFF];
    bool live[MV_OFF];
#pragma unroll
    for (int k = 0; k < MV_OFF; ++k) {
        const unsigned long long i = i0 + k * MV_THREADS;
        live[k] = i < span;
        const uint32_t r = (uint32_t)(i / cpr);
        row[k] = p.row0[lo] + r;
        off[k] = (size_t)row[k] * p.g.row_stride + (size_t)(i - (unsigned long long)r * cpr) * VEC;
    }
    T tmp[MV_OFF];
    const uint32_t e = p.comp[lo + 1];
    for (uint32_t j0 = p.comp[lo]; j0 < e; j0 += MV_BAT) {
        T v[MV_BAT][MV_OFF];
#pragma unroll
        for (int j = 0; j < MV_BAT; ++j)
            if (j0 + j < e) {
                const MoveIns in = p.ins[j0 + j];
#pragma unroll
                for (int k = 0; k < MV_OFF; ++k) {
                    if (in.src == MOVE_TMP) {
                        v[j][k] = tmp[k];
                    } else if (live[k] && row[k] - in.start < in.len) {
                        if (j > 0 && p.ins[j0 + j - 1].src == in.src && p.ins[j0 + j - 1].start == in.start &&
                            p.ins[j0 + j - 1].len == in.len)
                            v[j][k] = v[j > 0 ? j - 1 : 0][k];
                        else
                            v[j][k] = *(const T*)(base + (size_t)in.src * p.g.slot_stride + off[k]);
                    }
                    if (in.dst == MOVE_TMP) tmp[k] = v[j][k];
                }
            }
#pragma unroll
        for (int j = 0; j < MV_BAT; ++j)
            if (j0 + j < e) {
                const MoveIns in = p.ins[j0 + j];
                if (in.dst == MOVE_TMP) continue;
#pragma unroll
                for (int k = 0; k < MV_OFF; ++k)
                    if (live[k] && row[k] - in.start < in.len)
                        *(T*)(base + (size_t)in.dst * p.g.slot_stride + off[k]) = v[j][k];
            }
    }
}

template <int CAP>
static cudaError_t launch_cap(const MoveGeom& g, const MoveIns* ins, const uint32_t* comp, int n_comp,
                              cudaStream_t s) {
    static thread_local MoveProg<CAP> p;  // tens of KB at the large capacity: not on the stack
    p.g = g;
    p.n_comp = n_comp;
    memcpy(p.ins, ins, comp[n_comp] * sizeof(MoveIns));
    memcpy(p.comp, comp, (n_comp + 1) * sizeof(uint32_t));
    // the widest access that every address allows
    size_t all = g.slot_stride | g.outer_stride | g.row_stride | g.row_bytes;
    for (int i = 0; i < g.n_base; ++i) all |= (size_t)g.base[i];
    const int vec = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    unsigned long long blocks = 0;
    for (int c = 0; c < n_comp; ++c) {
        uint32_t r0 = 0xffffffffu, r1 = 0;
        for (uint32_t j = comp[c]; j < comp[c + 1]; ++j) {
            r0 = ins[j].start < r0 ? ins[j].start : r0;
            r1 = ins[j].start + ins[j].len > r1 ? ins[j].start + ins[j].len : r1;
        }
        p.row0[c] = r0;
        p.rows[c] = r1 - r0;
        p.block[c] = (uint32_t)blocks;
        const unsigned long long span = (unsigned long long)(r1 - r0) * (g.row_bytes / vec);
        blocks += (span + MV_THREADS * MV_OFF - 1) / (MV_THREADS * MV_OFF) * g.n_outer * g.n_base;
        if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
    }
    p.block[n_comp] = (uint32_t)blocks;
    if (blocks == 0) return cudaSuccess;
    switch (vec) {
        case 16: k_kv_move<16, CAP><<<(unsigned)blocks, MV_THREADS, 0, s>>>(p); break;
        case 8: k_kv_move<8, CAP><<<(unsigned)blocks, MV_THREADS, 0, s>>>(p); break;
        case 4: k_kv_move<4, CAP><<<(unsigned)blocks, MV_THREADS, 0, s>>>(p); break;
        case 2: k_kv_move<2, CAP><<<(unsigned)blocks, MV_THREADS, 0, s>>>(p); break;
        default: k_kv_move<1, CAP><<<(unsigned)blocks, MV_THREADS, 0, s>>>(p); break;
    }
    return cudaGetLastError();
}

// Up to 64 moves (a batch's slots) fit a small parameter block; the large one
// holds MOVE_MAX moves in 20 KB of kernel parameters.
cudaError_t launch_kv_move(const MoveGeom& g, const MoveIns* ins, const uint32_t* comp, int n_comp, cudaStream_t s) {
    const uint32_t n = comp[n_comp];
    if (n_comp <= 64 && n <= 96) return launch_cap<64>(g, ins, comp, n_comp, s);
    if (n_comp <= MOVE_MAX && n <= MOVE_MAX + MOVE_MAX / 2) return launch_cap<MOVE_MAX>(g, ins, comp, n_comp, s);
    return cudaErrorInvalidValue;
}

}  // namespace talos
