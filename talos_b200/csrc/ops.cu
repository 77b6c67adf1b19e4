// ops.cu -- the entry points of the batch operators in include/talos_cuda.h:
// checks of their arguments, the plan of a call's moves, the launches.
#include <string.h>

#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

#include "ops.cuh"
#include "status.cuh"

using namespace talos;

namespace {

// The call's device made current, and the caller's again at the end.
struct OnDevice {
    int before = -1;
    cudaError_t err;
    explicit OnDevice(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

talos_status on_device(const OnDevice& d, int device) {
    if (d.err == cudaSuccess) return TALOS_OK;
    cudaGetLastError();
    return set_err(d.err == cudaErrorInvalidDevice ? TALOS_ERR_INVALID_ARG : TALOS_ERR_CUDA, "device %d: %s", device,
                   cudaGetErrorString(d.err));
}

bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

}  // namespace

talos_status talos::ops_configured(int device) {
    static std::mutex mu;
    static bool done[64];
    if (device < 0 || device >= 64) return set_err(TALOS_ERR_INVALID_ARG, "device %d", device);
    std::lock_guard<std::mutex> lk(mu);
    if (done[device]) return TALOS_OK;
    CK(sample_configure());
    CK(attn_shared_configure());
    done[device] = true;
    return TALOS_OK;
}

// ------------------------------------------------------------------ token choice

extern "C" talos_status talos_sample_dev(const talos_sample_args* a, void* stream) {
    if (!a) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    const int es = dtype_bytes(a->type);
    if (!es) return set_err(TALOS_ERR_UNSUPPORTED, "logits of type %d (F32, F16 or BF16)", a->type);
    if (a->n == 0) return TALOS_OK;
    if (!a->logits || !a->u || !a->tokens) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if (a->vocab == 0 || a->vocab > (uint32_t)SAMPLE_MAX_VOCAB)
        return set_err(TALOS_ERR_INVALID_ARG, "%u logits per row (1 .. %d)", a->vocab, SAMPLE_MAX_VOCAB);
    if (a->n > 1u << 24) return set_err(TALOS_ERR_INVALID_ARG, "%u rows (at most %u)", a->n, 1u << 24);
    if (a->n > 1 && a->row_stride < a->vocab)
        return set_err(TALOS_ERR_INVALID_ARG, "rows %zu elements apart hold %u logits", a->row_stride, a->vocab);
    if (!aligned(a->logits, es) || !aligned(a->u, 4) || !aligned(a->tokens, 4) || !aligned(a->probs, 4) ||
        !aligned(a->temperature_dev, 4) || !aligned(a->top_k_dev, 4) || !aligned(a->top_p_dev, 4) ||
        !aligned(a->min_p_dev, 4))
        return set_err(TALOS_ERR_INVALID_ARG, "a pointer is not aligned to its element");
    if (!a->top_k_dev && a->top_k < 0) return set_err(TALOS_ERR_INVALID_ARG, "top_k %d", a->top_k);
    OnDevice d(a->device);
    TRY(on_device(d, a->device));
    TRY(ops_configured(a->device));
    SampleArgs k{};
    k.logits = a->logits;
    k.stride = a->n > 1 ? a->row_stride : a->vocab;
    k.n = (int)a->n, k.vocab = (int)a->vocab;
    k.u = a->u;
    k.temperature_dev = a->temperature_dev, k.top_k_dev = a->top_k_dev;
    k.top_p_dev = a->top_p_dev, k.min_p_dev = a->min_p_dev;
    k.temperature = a->temperature, k.top_k = a->top_k, k.top_p = a->top_p, k.min_p = a->min_p;
    k.tokens = a->tokens, k.probs = a->probs;
    CK(launch_sample(k, a->type, sm_count_dev(a->device), (cudaStream_t)stream));
    return TALOS_OK;
}

extern "C" talos_status talos_sample(const float* logits, size_t n, float u, float temperature, int32_t top_k,
                                     float top_p, float min_p, uint32_t* index_out, float* prob_out) {
    if (!logits || !index_out) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if (n == 0 || n > (size_t)SAMPLE_MAX_VOCAB)
        return set_err(TALOS_ERR_INVALID_ARG, "%zu logits (1 .. %d)", n, SAMPLE_MAX_VOCAB);
    if (top_k < 0) return set_err(TALOS_ERR_INVALID_ARG, "top_k %d", top_k);
    int dev = 0;
    CK(cudaGetDevice(&dev));
    float* mem = nullptr;  // logits, then u, token, probability
    CK(cudaMalloc(&mem, n * 4 + 12));
    int32_t token = -1;
    float prob = 0.f;
    cudaError_t e = cudaMemcpy(mem, logits, n * 4, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(mem + n, &u, 4, cudaMemcpyHostToDevice);
    talos_status st = TALOS_OK;
    if (e == cudaSuccess) {
        talos_sample_args a{};
        a.device = dev, a.type = TALOS_F32, a.n = 1, a.vocab = (uint32_t)n;
        a.logits = mem, a.row_stride = n, a.u = mem + n;
        a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
        a.tokens = (int32_t*)(mem + n + 1), a.probs = mem + n + 2;
        st = talos_sample_dev(&a, nullptr);
        if (st == TALOS_OK) e = cudaMemcpy(&token, a.tokens, 4, cudaMemcpyDeviceToHost);
        if (st == TALOS_OK && e == cudaSuccess) e = cudaMemcpy(&prob, a.probs, 4, cudaMemcpyDeviceToHost);
    }
    cudaFree(mem);
    TRY(st);
    if (e != cudaSuccess) return set_err(TALOS_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
    if (token < 0) return set_err(TALOS_ERR_INVALID_ARG, "no logit above -inf");
    *index_out = (uint32_t)token;
    if (prob_out) *prob_out = prob;
    return TALOS_OK;
}

// ------------------------------------------------------------------ attention over a shared prefix

extern "C" talos_status talos_attention_shared_work(int device, uint32_t n, uint32_t n_head, uint32_t n_head_kv,
                                                    size_t* out) {
    if (!out) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if (!n || n > 1024) return set_err(TALOS_ERR_INVALID_ARG, "%u sequences (1 .. 1024)", n);
    if (!n_head_kv || n_head % n_head_kv || !n_head || n_head / n_head_kv > 128)
        return set_err(TALOS_ERR_INVALID_ARG, "%u heads over %u kv heads (a multiple, at most 128 times)", n_head,
                       n_head_kv);
    *out = attn_shared_work_bytes((int)n, (int)(n_head / n_head_kv), sm_count_dev(device));
    return TALOS_OK;
}

extern "C" talos_status talos_attention_shared_dev(const talos_attention_shared_args* a, void* work, size_t work_bytes,
                                                   void* stream) {
    if (!a) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if (!attn_shared_types(a->q_type, a->kv_type))
        return set_err(TALOS_ERR_UNSUPPORTED, "queries of type %d with a cache of type %d", a->q_type, a->kv_type);
    if (a->n == 0) return TALOS_OK;
    size_t need = 0;
    TRY(talos_attention_shared_work(a->device, a->n, a->n_head, a->n_head_kv, &need));
    const int qs = dtype_bytes(a->q_type), ks = dtype_bytes(a->kv_type);
    if (!a->head_dim || a->head_dim > 128 || a->head_dim % (qs == 4 && ks == 4 ? 4 : 8))
        return set_err(TALOS_ERR_UNSUPPORTED, "head_dim %u (a multiple of 8, or of 4 with an f32 cache, up to 128)",
                       a->head_dim);
    if (!(a->scale >= 1e-30f && a->scale <= 1e30f)) return set_err(TALOS_ERR_INVALID_ARG, "scale %g", (double)a->scale);
    if (!a->q || !a->out || !a->lens || !work) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if ((a->prefix_len && (!a->k_prefix || !a->v_prefix)) || (a->n_slots && a->slot_len && (!a->k || !a->v)))
        return set_err(TALOS_ERR_INVALID_ARG, "NULL cache");
    if (work_bytes < need) return set_err(TALOS_ERR_INVALID_ARG, "workspace of %zu bytes, needs %zu", work_bytes, need);
    if (a->n_slots > 0x7fffffffu || !a->n_slots)
        return set_err(TALOS_ERR_INVALID_ARG, "%u slots", a->n_slots);
    const uint64_t spt = 128 / (a->n_head / a->n_head_kv);
    const uint64_t tiles = a->prefix_len / 64 + 1 + std::min<uint64_t>(a->n, spt) * (a->slot_len / 64 + 1ull);
    // the kernels count the tiles of a row tile over the kv heads, of a kv head over the row
    // tiles, a row tile's output elements and the second kernel's warps in 32 bits
    const uint64_t row_tiles = (a->n + spt - 1) / spt;
    if (tiles * std::max<uint64_t>(a->n_head_kv, row_tiles) > 0x3fffffffull || a->prefix_len > 0x3fffffffu ||
        a->slot_len > 0x3fffffffu)
        return set_err(TALOS_ERR_UNSUPPORTED, "prefix of %u and slots of %u positions for %u sequences", a->prefix_len,
                       a->slot_len, a->n);
    if (128ull * a->n_head_kv * a->head_dim > 0x3fffffffull || row_tiles * a->n_head_kv * 128 > 0x3fffffffull)
        return set_err(TALOS_ERR_UNSUPPORTED, "%u sequences of %u heads", a->n, a->n_head);
    AttnSharedArgs k{};
    // a dimension of one element (or none) has no stride to speak of
    auto st = [](size_t stride, uint32_t count) { return count > 1 ? stride : 0; };
    k.q_sn = st(a->q_stride_n, a->n), k.q_sh = st(a->q_stride_h, a->n_head);
    k.out_sn = st(a->out_stride_n, a->n), k.out_sh = st(a->out_stride_h, a->n_head);
    k.pre_st = st(a->prefix_stride_t, a->prefix_len);
    k.pre_sh = a->prefix_len ? st(a->prefix_stride_h, a->n_head_kv) : 0;
    if (a->slot_len) {
        k.slot_ss = st(a->slot_stride, a->n_slots), k.slot_st = st(a->slot_stride_t, a->slot_len);
        k.slot_sh = st(a->slot_stride_h, a->n_head_kv);
    }
    for (size_t x : {k.q_sn * qs, k.q_sh * qs, k.out_sn * qs, k.out_sh * qs, k.pre_st * ks, k.pre_sh * ks,
                     k.slot_ss * ks, k.slot_st * ks, k.slot_sh * ks})
        if (x % 16) return set_err(TALOS_ERR_INVALID_ARG, "a stride of %zu bytes (multiples of 16)", x);
    {  // the output's rows must not overlap
        const uint64_t cn = k.out_sn ? a->n : 1, ch = k.out_sh ? a->n_head : 1;
        const bool n_outer = k.out_sn >= k.out_sh;
        const uint64_t s0 = n_outer ? k.out_sh : k.out_sn, c0 = n_outer ? ch : cn, s1 = n_outer ? k.out_sn : k.out_sh;
        const bool apart = (a->n == 1 || k.out_sn) && (a->n_head == 1 || k.out_sh) && (c0 == 1 || s0 >= a->head_dim) &&
                           ((cn == 1 && ch == 1) || cn * ch == c0 || s1 >= s0 * (c0 - 1) + a->head_dim);
        if (!apart) return set_err(TALOS_ERR_INVALID_ARG, "the output's strides make its rows overlap");
    }
    for (const void* p : {a->q, (const void*)a->out, a->k_prefix, a->v_prefix, a->k, a->v, (const void*)work})
        if (!aligned(p, 16)) return set_err(TALOS_ERR_INVALID_ARG, "a pointer is not 16-byte aligned");
    if (!aligned(a->lens, 4) || !aligned(a->slots, 4))
        return set_err(TALOS_ERR_INVALID_ARG, "a pointer is not aligned to its element");
    OnDevice d(a->device);
    TRY(on_device(d, a->device));
    TRY(ops_configured(a->device));
    k.q = a->q, k.kp = a->k_prefix, k.vp = a->v_prefix, k.k = a->k, k.v = a->v, k.out = a->out;
    k.n = (int)a->n, k.n_kv = (int)a->n_head_kv, k.group = (int)(a->n_head / a->n_head_kv), k.hd = (int)a->head_dim;
    k.prefix = (int)a->prefix_len, k.n_slots = (int)a->n_slots, k.slot_len = (int)a->slot_len;
    k.lens = a->lens, k.slots = a->slots;
    k.scale = a->scale;
    CK(launch_attn_shared(k, a->q_type, a->kv_type, work, sm_count_dev(a->device), (cudaStream_t)stream));
    return TALOS_OK;
}

// ------------------------------------------------------------------ cache moves

namespace {

// Orders a call's moves for k_kv_move: per component of connected slots, every
// read of a slot before its write. A move is ready when no waiting move reads its
// destination; where none is ready the waiting moves form a cycle (each slot has
// one incoming move at most, so a component has one cycle at most), opened by
// setting one destination's rows aside.
void plan_moves(std::vector<talos_kv_copy> m, std::vector<MoveIns>& ins,
                std::vector<uint32_t>& comp) {
    std::vector<uint32_t> used;  // the slots that the moves touch, numbered 0 ..
    for (const auto& x : m) used.push_back(x.src), used.push_back(x.dst);
    std::sort(used.begin(), used.end());
    used.erase(std::unique(used.begin(), used.end()), used.end());
    auto id = [&](uint32_t s) { return (int)(std::lower_bound(used.begin(), used.end(), s) - used.begin()); };
    const int ns = (int)used.size();
    // moves by source, so that one slot's destinations follow one another
    std::stable_sort(m.begin(), m.end(), [](const talos_kv_copy& x, const talos_kv_copy& y) { return x.src < y.src; });
    const int n = (int)m.size();
    std::vector<int> src(n), dst(n), readers(ns, 0), into(ns, -1), root(ns);
    for (int i = 0; i < ns; ++i) root[i] = i;
    auto find = [&](int x) {
        while (root[x] != x) x = root[x] = root[root[x]];
        return x;
    };
    for (int i = 0; i < n; ++i) {
        src[i] = id(m[i].src), dst[i] = id(m[i].dst);
        ++readers[src[i]];
        into[dst[i]] = i;
        root[find(src[i])] = find(dst[i]);
    }
    std::vector<std::vector<int>> by_comp(ns);
    for (int i = 0; i < n; ++i) by_comp[find(src[i])].push_back(i);
    comp.push_back(0);
    for (const auto& c : by_comp) {
        if (c.empty()) continue;
        std::vector<int> ready;
        std::vector<char> done(n, 0);
        for (auto it = c.rbegin(); it != c.rend(); ++it)
            if (readers[dst[*it]] == 0) ready.push_back(*it);
        size_t left = c.size();
        std::vector<char> aside(n, 0);  // the move reads the rows set aside
        while (left) {
            if (ready.empty()) {
                int open = -1, reader = -1;
                for (int i : c)
                    if (!done[i]) open = i;
                for (int i : c)
                    if (!done[i] && src[i] == dst[open]) reader = i;
                ins.push_back(MoveIns{m[reader].src, MOVE_TMP, m[reader].start, m[reader].len});
                aside[reader] = 1;
                readers[src[reader]] = 0;
                ready.push_back(open);
                continue;
            }
            const int i = ready.back();
            ready.pop_back();
            ins.push_back(MoveIns{aside[i] ? MOVE_TMP : m[i].src, m[i].dst, m[i].start, m[i].len});
            done[i] = 1;
            --left;
            if (!aside[i] && --readers[src[i]] == 0) {
                const int w = into[src[i]];
                if (w >= 0 && !done[w]) ready.push_back(w);
            }
        }
        comp.push_back((uint32_t)ins.size());
    }
}

// Rows are disjoint when, from the smallest stride to the largest, each steps
// over all that lies below it.
struct MoveDim {
    size_t stride, count;
};
bool disjoint(const talos_kv_slots& g, MoveDim (&d)[3]) {
    d[0] = {g.row_stride, g.n_rows}, d[1] = {g.outer_stride, g.n_outer}, d[2] = {g.slot_stride, g.n_slots};
    std::sort(d, d + 3, [](const MoveDim& x, const MoveDim& y) { return x.stride < y.stride; });
    size_t span = g.row_bytes;
    for (const MoveDim& x : d) {
        if (x.count <= 1) continue;
        if (x.stride < span) return false;
        if (x.stride > ((size_t)1 << 62) / x.count) return false;
        span = x.stride * (x.count - 1) + span;
    }
    return true;
}
// Whether a row of one array lies over one of another whose base is `off` bytes away: some
// difference of indexes brings them together. The stride of a (disjoint) geometry's largest
// dimension exceeds all that the others reach, so its difference is one of three.
bool rows_meet(int64_t off, const MoveDim* d, int n, int64_t row_bytes) {
    if (n == 0) return off < row_bytes && -off < row_bytes;
    const MoveDim& x = d[n - 1];
    if (x.count <= 1) return rows_meet(off, d, n - 1, row_bytes);
    const int64_t s = (int64_t)x.stride, most = (int64_t)x.count - 1, k0 = -(off / s);
    for (int64_t k = std::max(k0 - 1, -most); k <= std::min(k0 + 1, most); ++k)
        if (rows_meet(off + k * s, d, n - 1, row_bytes)) return true;
    return false;
}

}  // namespace

extern "C" talos_status talos_kv_move_dev(const talos_kv_slots* g, const talos_kv_copy* moves, size_t n, void* stream) {
    if (!g || (!moves && n)) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    if (g->n_base < 1 || g->n_base > MOVE_MAX_BASE)
        return set_err(TALOS_ERR_INVALID_ARG, "%d arrays (1 .. %d)", g->n_base, MOVE_MAX_BASE);
    if (!g->base) return set_err(TALOS_ERR_INVALID_ARG, "NULL argument");
    for (int i = 0; i < g->n_base; ++i) {
        if (!g->base[i]) return set_err(TALOS_ERR_INVALID_ARG, "array %d is NULL", i);
        for (int j = 0; j < i; ++j)
            if (g->base[i] == g->base[j]) return set_err(TALOS_ERR_INVALID_ARG, "arrays %d and %d are the same", j, i);
    }
    if (n > (size_t)MOVE_MAX) return set_err(TALOS_ERR_INVALID_ARG, "%zu moves (at most %d)", n, MOVE_MAX);
    if (!g->row_bytes || !g->n_outer || g->row_bytes > 0xffffffffu)
        return set_err(TALOS_ERR_INVALID_ARG, "rows of %zu bytes in %u planes", g->row_bytes, g->n_outer);
    MoveDim dims[3];
    if (!disjoint(*g, dims)) return set_err(TALOS_ERR_INVALID_ARG, "the strides make rows overlap");
    for (int i = 0; i < g->n_base; ++i)
        for (int j = 0; j < i; ++j)
            if (rows_meet((int64_t)((uintptr_t)g->base[i] - (uintptr_t)g->base[j]), dims, 3, (int64_t)g->row_bytes))
                return set_err(TALOS_ERR_INVALID_ARG, "rows of arrays %d and %d overlap", j, i);
    try {
        std::vector<talos_kv_copy> live;
        std::vector<uint32_t> dsts;
        for (size_t i = 0; i < n; ++i) {
            const talos_kv_copy& m = moves[i];
            if (m.src >= g->n_slots || m.dst >= g->n_slots)
                return set_err(TALOS_ERR_INVALID_ARG, "move %zu: slot %u -> %u of %u", i, m.src, m.dst, g->n_slots);
            if ((uint64_t)m.start + m.len > g->n_rows)
                return set_err(TALOS_ERR_INVALID_ARG, "move %zu: rows %u .. %llu of %u", i, m.start,
                               (unsigned long long)m.start + m.len, g->n_rows);
            dsts.push_back(m.dst);
            if (m.src != m.dst && m.len) live.push_back(m);
        }
        std::sort(dsts.begin(), dsts.end());
        for (size_t i = 1; i < dsts.size(); ++i)
            if (dsts[i] == dsts[i - 1])
                return set_err(TALOS_ERR_INVALID_ARG, "slot %u is the destination of two moves", dsts[i]);
        if (live.empty()) return TALOS_OK;
        std::vector<MoveIns> ins;
        std::vector<uint32_t> comp;
        plan_moves(std::move(live), ins, comp);
        MoveGeom k{};
        for (int i = 0; i < g->n_base; ++i) k.base[i] = (uint8_t*)g->base[i];
        k.n_base = g->n_base;
        k.n_outer = g->n_outer;
        k.slot_stride = g->slot_stride, k.outer_stride = g->n_outer > 1 ? g->outer_stride : 0;
        k.row_stride = g->row_stride, k.row_bytes = g->row_bytes;
        OnDevice d(g->device);
        TRY(on_device(d, g->device));
        const cudaError_t e = launch_kv_move(k, ins.data(), comp.data(), (int)comp.size() - 1, (cudaStream_t)stream);
        if (e == cudaErrorInvalidValue) return set_err(TALOS_ERR_UNSUPPORTED, "more rows than one launch takes");
        CK(e);
        return TALOS_OK;
    } catch (const std::bad_alloc&) {
        return set_err(TALOS_ERR_OOM, "host memory for the plan of %zu moves", n);
    }
}
