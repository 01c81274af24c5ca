// k_kv_attn.cu — attention of rows over a KV cache (kv.cuh): causal or a tree of drafts, within a sliding window, the
// first `sinks` positions always visible.
//
// out[t] = sum_p softmax_p(scale q_t . k_p) v_p over the visible positions p: p <= pos + t, and with a window also
// p > pos + t - window or p < sinks. Drafts (a parent for each row): row t stands at position pos + depth(t) and sees
// the committed positions and, of the drafts, its ancestors and itself. A row that sees nothing gives zeros.
//
// The simple form: one warp per (slot, row, head), a key at a time, lane i holding dims i, i + 32, …
#include "kv.cuh"

namespace ocr {

template <int TYPE>
__device__ __forceinline__ float kv_value(const uint8_t* q, const __half* s, size_t row, int d, int i) {
    if (TYPE == KV_F16) return __half2float(reinterpret_cast<const __half*>(q)[row * d + i]);
    const float scale = __half2float(s[row * (d / KV_BLOCK) + i / KV_BLOCK]);
    if (TYPE == KV_Q8_0) return (float)reinterpret_cast<const int8_t*>(q)[row * d + i] * scale;
    const int j = i % KV_BLOCK;
    const uint8_t w = q[row * (d / 2) + i / KV_BLOCK * 16 + j % 16];
    return ((float)(j < 16 ? w & 15 : w >> 4) - 8.0f) * scale;
}

template <int TYPE, int D, class T>
__global__ void __launch_bounds__(128) k_kv_attn_simple(KvAttnArgs a) {
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    const int lane = threadIdx.x & 31;
    const long w = ((long)blockIdx.x * 128 + threadIdx.x) >> 5;
    const long per_slot = (long)a.r.T * a.n_head;
    const int b = (int)(w / per_slot);
    if (b >= c.n_slot) return;
    const int t = (int)(w % per_slot) / a.n_head, h = (int)(w % a.n_head);
    const T* q = static_cast<const T*>(a.q) + b * a.q_slot + t * a.q_row + h * a.q_head;
    T* out = static_cast<T*>(a.out) + b * a.o_slot + t * a.o_row + h * a.o_head;
    const int n = a.r.rows(c, b, a.err);
    if (t >= n) {
        for (int i = lane; i < D; i += 32) out[i] = (T)0.0f;
        return;
    }
    const int pos = a.r.pos[b];
    const int32_t* parent = a.parent ? a.parent + (size_t)b * a.r.T : nullptr;
    uint64_t anc = 0;
    int at = pos + t;
    if (parent) {
        int depth = -1;
        for (int i = t; i >= 0; depth++) {
            anc |= 1ull << i;
            const int p = parent[i];
            if (p >= i || p < -1) {
                dev_error(a.err, DEV_BAD_INDEX);
                depth++;
                break;
            }
            i = p;
        }
        at = pos + depth;
    }
    float qv[D / 32], o[D / 32] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; i++) qv[i] = (float)q[lane + 32 * i] * a.scale;
    const int lo = c.window ? max(0, at - c.window + 1) : 0;
    const int end = pos + t + 1;
    for (int p = 0; p < end; p++) {
        if (p == min(c.sinks, lo) && p < lo) p = min(lo, pos);
        int where = p;
        if (parent && p >= pos) {
            if (!((anc >> (p - pos)) & 1)) continue;
            where = pos - 1;
            for (int i = p - pos; i >= 0; where++) i = parent[i] < i ? parent[i] : -1;
        }
        if (c.window && where <= at - c.window && where >= c.sinks) continue;
        const size_t row = kv_index(c, b, h / (a.n_head / c.n_kv), kv_row(c, p));
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) s += qv[i] * kv_value<TYPE>(c.k, c.ks, row, D, lane + 32 * i);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), f = expf(m - mn), e = mn == -INFINITY ? 0.0f : expf(s - mn);
        l = (m == -INFINITY ? 0.0f : l * f) + e;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
            o[i] = (m == -INFINITY ? 0.0f : o[i] * f) + e * kv_value<TYPE>(c.v, c.vs, row, D, lane + 32 * i);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < D / 32; i++) out[lane + 32 * i] = (T)(l == 0.0f ? 0.0f : o[i] / l);
}

template <int TYPE, int D>
static cudaError_t launch_d(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    const long warps = (long)a.c.n_slot * a.r.T * a.n_head;
    const dim3 grid((unsigned)((warps + 3) / 4));
    return a.half ? kv_launch(k_kv_attn_simple<TYPE, D, __half>, grid, 128, 0, st, pdl, a)
                  : kv_launch(k_kv_attn_simple<TYPE, D, float>, grid, 128, 0, st, pdl, a);
}
template <int TYPE>
static cudaError_t launch_type(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    return a.c.d == 128 ? launch_d<TYPE, 128>(st, a, pdl) : launch_d<TYPE, 64>(st, a, pdl);
}
static cudaError_t launch_simple(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    switch (a.c.type) {
        case KV_F16: return launch_type<KV_F16>(st, a, pdl);
        case KV_Q8_0: return launch_type<KV_Q8_0>(st, a, pdl);
        default: return launch_type<KV_Q4_0>(st, a, pdl);
    }
}

cudaError_t launch_kv_attention(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    return a.r.T * (a.n_head / a.c.n_kv) <= 32 ? launch_kv_attention_few(st, a, pdl) : launch_simple(st, a, pdl);
}
size_t kv_attention_work_bytes(const KvAttnArgs& a) { return 4096 + (size_t)a.num_sms * 2 * 4 * (128 * 8 + 16) * 4; }

}  // namespace ocr
