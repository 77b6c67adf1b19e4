// kvmove.cu -- rows moved between cache slots on B200 (sm_100a): a prompt
// copied (forked) into other slots, live slots compacted to the front.
//
// A move copies rows [start, start + len) of slot src to slot dst, in every
// array (K, V) and layer. The moves of a call are simultaneous: every read sees
// the data from before the call. The host orders them so that each slot is read
// by all its readers before it is overwritten, and groups them into components
// that touch disjoint slots; a cycle of slots keeps one chunk aside (MOVE_TMP).
// A thread takes offsets of a component (array, layer, row, 16 bytes of the
// row) and carries out all of the component's moves at each of them, so the
// order between them is its own program order: no barrier, no second buffer,
// and a slot copied to many others is read once.
//
// Bound: HBM. Each source row is read once, each destination row written once.
// What carries it is warps in flight (one 16-byte load a thread, 32 registers, 8
// blocks an SM) and long runs within a slot. One prompt of 512 rows into 31 slots
// (1.07 GB with 8 layers of 2 x 4 KB rows): 173 us, 6.2 TB/s; 40 slots of up to 1000 rows
// moved to the front (1.64 GB, f16): 246 us, 6.7 TB/s. With 16 loads a thread in
// flight (199 registers, one block an SM) they took 298 and 870 us.
#include <string.h>

#include "ops.cuh"

namespace talos {

constexpr int MV_THREADS = 256;

template <int CAP>
struct MoveProg {
    MoveGeom g;
    int n_comp, iter;          // iter: offsets a thread takes
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

template <int VEC, int CAP>
__global__ void __launch_bounds__(MV_THREADS, 8) k_kv_move(const __grid_constant__ MoveProg<CAP> p) {
    using T = typename MvWord<VEC>::T;
    int lo = 0, hi = p.n_comp;  // the component of this block
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.block[mid] <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const uint32_t cpr = (uint32_t)(p.g.row_bytes / VEC);  // chunks per row
    const unsigned long long span = (unsigned long long)p.rows[lo] * cpr;
    const uint32_t per_block = MV_THREADS * (uint32_t)p.iter;
    const uint32_t per_outer = (uint32_t)((span + per_block - 1) / per_block);
    const uint32_t b = blockIdx.x - p.block[lo];
    const uint32_t outer = b / per_outer;  // (array, layer)
    uint8_t* base = p.g.base[outer / p.g.n_outer] + (size_t)(outer % p.g.n_outer) * p.g.outer_stride;
    const unsigned long long i0 = (unsigned long long)(b % per_outer) * per_block + threadIdx.x;
    const uint32_t e = p.comp[lo + 1];
    if (p.iter == 1) {
        const uint32_t r = span <= 0xffffffffull ? (uint32_t)i0 / cpr : (uint32_t)(i0 / cpr);
        const uint32_t row = p.row0[lo] + r;
        if (i0 >= span) return;
        uint8_t* at = base + (size_t)row * p.g.row_stride + (size_t)(i0 - (unsigned long long)r * cpr) * VEC;
        T v = {}, tmp = {};
        MoveIns last{MOVE_TMP, MOVE_TMP, 0, 0};
#pragma unroll 4
        for (uint32_t j = p.comp[lo]; j < e; ++j) {
            const MoveIns in = p.ins[j];
            if (row - in.start < in.len) {
                if (in.src == MOVE_TMP) v = tmp;
                else if (in.src != last.src || in.start != last.start || in.len != last.len)
                    v = *(const T*)(at + (size_t)in.src * p.g.slot_stride);
                if (in.dst == MOVE_TMP) tmp = v;
                else *(T*)(at + (size_t)in.dst * p.g.slot_stride) = v;
            }
            last = in;
        }
        return;
    }
    for (uint32_t j = p.comp[lo]; j < e; ++j) {
        const MoveIns in = p.ins[j];
#pragma unroll 1
        for (int it = 0; it < p.iter; ++it) {
            const unsigned long long i = i0 + (uint32_t)it * MV_THREADS;
            const uint32_t r = span <= 0xffffffffull ? (uint32_t)i / cpr : (uint32_t)(i / cpr);
            const uint32_t row = p.row0[lo] + r;
            if (i >= span || row - in.start >= in.len) continue;
            uint8_t* at = base + (size_t)row * p.g.row_stride + (size_t)(i - (unsigned long long)r * cpr) * VEC;
            *(T*)(at + (size_t)in.dst * p.g.slot_stride) = *(const T*)(at + (size_t)in.src * p.g.slot_stride);
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
    // Offsets of a thread: one where a source is copied to several slots in a row or a chunk
    // is kept aside; else up to 8, so that a block reads and writes 32 KB of a slot at a
    // stretch (40 slots: 382 -> 267 us; a fork, reading its source for each copy, would take
    // 245 instead of 173), as long as the blocks fill 148 SMs twice.
    bool one = false;
    unsigned long long blocks = 0;
    for (int c = 0; c < n_comp; ++c) {
        uint32_t r0 = 0xffffffffu, r1 = 0;
        for (uint32_t j = comp[c]; j < comp[c + 1]; ++j) {
            r0 = ins[j].start < r0 ? ins[j].start : r0;
            r1 = ins[j].start + ins[j].len > r1 ? ins[j].start + ins[j].len : r1;
            one |= ins[j].src == MOVE_TMP || ins[j].dst == MOVE_TMP || (j > comp[c] && ins[j].src == ins[j - 1].src);
        }
        p.row0[c] = r0;
        p.rows[c] = r1 - r0;
    }
    for (p.iter = one ? 1 : 8;; p.iter /= 2) {
        const unsigned long long per_block = (unsigned long long)MV_THREADS * p.iter;
        blocks = 0;
        for (int c = 0; c < n_comp; ++c) {
            p.block[c] = (uint32_t)blocks;
            blocks += (p.rows[c] * (unsigned long long)(g.row_bytes / vec) + per_block - 1) / per_block * g.n_outer *
                      g.n_base;
            if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
        }
        if (p.iter == 1 || blocks >= 2 * 8 * 148) break;
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
