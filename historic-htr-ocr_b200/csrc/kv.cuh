// kv.cuh — one layer's KV cache in f16, q8_0 or q4_0, as the kernels see it (ocr_kv_cache, include/ocr_cuda.h), and the
// launchers of the operators over it: rows written, read back and moved (k_kv_cache.cu), the attentions (k_kv_attn.cu,
// k_kv_attn_one.cu, k_kv_attn_tc.cu).
//
// Layout, per tensor (K and V alike): quants [n_slot][n_kv][n_rows][row bytes], scales [n_slot][n_kv][n_rows][d / 32]
// f16. Offsets are 64-bit: a long cache passes 2^31 bytes. A position p of a slot lives in row p; in a ring cache the
// rows from `sinks` on are used round and round, so position p >= sinks lives in sinks + (p - sinks) % (n_rows - sinks).
#pragma once

#include "common.cuh"

namespace ocr {

constexpr int KV_F16 = 1, KV_Q4_0 = 2, KV_Q8_0 = 8;  // ocr_kv_cache.type (ggml's numbers)
constexpr int KV_BLOCK = 32;                         // values that share a scale
constexpr int KV_TICKETS = 4096;                     // bytes of the workspace before the partial results: a ticket per CTA
constexpr int KV_TREE_MAX = 64;                      // drafts of one tree: an ancestor set is one 64-bit word

__host__ __device__ constexpr int kv_row_bytes(int type, int d) {
    return type == KV_F16 ? 2 * d : type == KV_Q8_0 ? d : d / 2;
}

struct KvView {
    uint8_t *k, *v;
    __half *ks, *vs;  // scales (null for f16)
    int type, n_slot, n_kv, d, n_rows, window, sinks, ring;
};

// rows of vectors: element (slot b, row t, head h, i) at p + b * slot + t * row + h * head + i (strides in elements)
template <class T>
struct RowsT {
    T* p;
    long slot, row, head;
    __device__ __forceinline__ T* at(int b, int t, int h) const { return p + b * slot + t * row + h * head; }
};

// the rows of one call: T of every slot from position pos[b] on, n[b] of them in use (null: all)
struct KvRange {
    const int32_t* pos;
    const int32_t* n;
    int T;
    // rows of slot b in use: 0 for an idle slot (pos < 0); a slot whose rows do not fit the cache is flagged and idle
    __device__ __forceinline__ int rows(const KvView& c, int b, int* err) const {
        const int p = pos[b];
        if (p < 0) return 0;
        const int m = n ? min(max(n[b], 0), T) : T;
        const bool fits = c.ring ? (long)p + m <= 0x7fffffffL : (long)p + m <= (long)c.n_rows;
        if (!fits) dev_error(err, DEV_BAD_POS);
        return fits ? m : 0;
    }
};

__device__ __forceinline__ int kv_row(const KvView& c, int p) {
    return c.ring && p >= c.sinks ? c.sinks + (p - c.sinks) % (c.n_rows - c.sinks) : p;
}
// the row's index in the [n_slot][n_kv][n_rows] order of the quants and the scales
__device__ __forceinline__ size_t kv_index(const KvView& c, int b, int h, int row) {
    return ((size_t)b * c.n_kv + h) * c.n_rows + row;
}

// ---- launchers ----
struct KvMoveArgs {
    KvView c;
    KvRange r;
    void *k, *v;  // f32 or f16 rows
    int half;
    long k_slot, k_row, k_head, v_slot, v_row, v_head;
    int* err;
};
cudaError_t launch_kv_write(cudaStream_t st, const KvMoveArgs& a, bool pdl);
cudaError_t launch_kv_read(cudaStream_t st, const KvMoveArgs& a, bool pdl);

constexpr int KV_KEEP_LAYERS = 64;  // layers of one launch
struct KvKeepArgs {
    KvView c;  // the shape shared by every layer
    struct {
        uint8_t *k, *v;
        __half *ks, *vs;
    } layer[KV_KEEP_LAYERS];
    int n_layer, T;
    const int32_t *pos, *path, *n;
    int* err;
};
cudaError_t launch_kv_keep(cudaStream_t st, const KvKeepArgs& a, bool pdl);

struct KvAttnArgs {
    KvView c;
    KvRange r;
    const int32_t* parent;  // the drafts' parents [n_slot][T] (null: rows in order)
    const void* q;
    void* out;
    int half, n_head;
    long q_slot, q_row, q_head, o_slot, o_row, o_head;
    float scale;
    void* work;  // partial results and tickets
    int num_sms;
    int* err;
};
// the call for slots b … b + n - 1 alone
inline KvAttnArgs kv_slots(const KvAttnArgs& all, int b, int n) {
    KvAttnArgs a = all;
    const size_t rows = (size_t)b * a.c.n_kv * a.c.n_rows, bytes = rows * kv_row_bytes(a.c.type, a.c.d);
    a.c.n_slot = n;
    a.c.k += bytes, a.c.v += bytes;
    if (a.c.ks) a.c.ks += rows * (a.c.d / KV_BLOCK), a.c.vs += rows * (a.c.d / KV_BLOCK);
    a.r.pos += b;
    if (a.r.n) a.r.n += b;
    if (a.parent) a.parent += (size_t)b * a.r.T;
    const long item = a.half ? 2 : 4;
    a.q = static_cast<const char*>(a.q) + b * a.q_slot * item;
    a.out = static_cast<char*>(a.out) + b * a.o_slot * item;
    return a;
}
cudaError_t launch_kv_attention(cudaStream_t st, const KvAttnArgs& a, bool pdl);
// (row, query head) pairs of a kv head up to which k_kv_attn_one.cu serves a quantised cache: with 2, 32 slots of some 3100
// keys in q8_0 take 55 us there and 73 in k_kv_attn.cu, in a q4_0 ring of 1028 keys 25 and 34. Its digits take
// four columns of eight a pair, so two pairs are what one product holds.
constexpr int KV_ONE_ROWS = 2;
cudaError_t launch_kv_attention_one(cudaStream_t st, const KvAttnArgs& a, bool pdl);
cudaError_t launch_kv_attention_many(cudaStream_t st, const KvAttnArgs& a, bool pdl);
// the bytes of the workspace that any call needs
size_t kv_attention_few_work(int num_sms);
size_t kv_attention_many_work(int num_sms);
size_t kv_attention_work_bytes(int num_sms);
long kv_attention_many_rows();
int kv_attention_many_slots(const KvAttnArgs& a);

// a launch that may start while its predecessor on the stream still runs: the kernel calls pdl_wait() before it
// touches memory
template <class... P, class... A>
cudaError_t kv_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool pdl, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}

}  // namespace ocr
