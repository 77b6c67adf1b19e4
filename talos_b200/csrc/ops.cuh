// ops.cuh -- launch interface of the device operators for many sequences that
// start from one prompt: the choice of tokens (sample.cu), moves between cache
// slots (kvmove.cu), attention over a shared prefix (attn_shared.cu).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace talos {

// Element types of device arrays (ggml tags).
enum DType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 30 };
inline int dtype_bytes(int t) { return t == DT_F32 ? 4 : (t == DT_F16 || t == DT_BF16) ? 2 : 0; }

// ---------------------------------------------------------------- token choice

struct SampleArgs {
    const void* logits;  // [n][stride] of type
    size_t stride;       // elements between rows
    int n, vocab;
    const float* u;      // [n] in [0, 1)
    // per-row settings, or (null) one value for every row
    const float* temperature_dev;
    const int32_t* top_k_dev;
    const float* top_p_dev;
    const float* min_p_dev;
    float temperature;
    int32_t top_k;
    float top_p, min_p;
    int32_t* tokens;  // [n]
    float* probs;     // [n] or null
    const int* n_dev;  // or null: rows in device memory (n is then their largest number)
};
constexpr int SAMPLE_MAX_VOCAB = 1 << 20;
cudaError_t sample_configure();  // once per device, on the current one
cudaError_t launch_sample(const SampleArgs& a, int type, int sms, cudaStream_t s);

// ---------------------------------------------------------------- cache moves

constexpr int MOVE_MAX = 512;  // moves of one call
constexpr int MOVE_MAX_BASE = 8;
struct MoveGeom {
    uint8_t* base[MOVE_MAX_BASE];
    int n_base;
    uint32_t n_outer;
    size_t slot_stride, outer_stride, row_stride;  // bytes
    size_t row_bytes;
};
struct MoveIns {
    uint32_t src, dst, start, len;  // src / dst may be MOVE_TMP
};
constexpr uint32_t MOVE_TMP = 0xffffffffu;
// ins: ordered so that every read of a slot precedes its write; comp[c] .. comp[c+1]
// are the instructions of component c (components touch disjoint slots).
cudaError_t launch_kv_move(const MoveGeom& g, const MoveIns* ins, const uint32_t* comp, int n_comp, cudaStream_t s);

// ---------------------------------------------------------------- attention over a shared prefix

struct AttnSharedArgs {
    // element strides: s*n sequences, *h heads, *t positions, *s slots
    const void* q;
    size_t q_sn, q_sh;
    const void *kp, *vp;  // prefix
    size_t pre_st, pre_sh;
    const void *k, *v;    // the sequences' slots
    size_t slot_ss, slot_st, slot_sh;
    void* out;
    size_t out_sn, out_sh;
    int n, n_kv, group, hd;
    int prefix, n_slots, slot_len;
    const int32_t* lens;   // suffix rows of each sequence
    const int32_t* slots;  // its slot (null: sequence i in slot i)
    float scale;
    // batched steps (f32 queries and cache): the sequence count and the prefix length in device memory (n and
    // prefix are then their largest values), positions instead of lengths (the
    // suffix has pos + 1 - prefix rows), suffix rows stored from row `prefix` of
    // the slot (slot_row0 = 1), error bits for a wait that ran out
    const int* n_dev;
    const uint32_t* prefix_dev;
    const uint32_t* pos;
    int slot_row0;
    uint32_t* error;
    // set by launch_attn_shared
    int whole;
    float2* part_ml;
    float4* part_o;
    int* plan;
};
bool attn_shared_types(int q_type, int kv_type);
cudaError_t attn_shared_configure();  // once per device, on the current one
size_t attn_shared_work_bytes(int n, int group, int sms);
// group <= 128, hd <= 128; work: attn_shared_work_bytes, 16-byte aligned
cudaError_t launch_attn_shared(AttnSharedArgs a, int q_type, int kv_type, void* work, int sms, cudaStream_t s);

}  // namespace talos
