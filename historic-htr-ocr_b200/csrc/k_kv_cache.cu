// k_kv_cache.cu — rows of keys and values quantised into a KV cache as they are written, read back as values, and the
// rows of an accepted path of drafts moved together.
//
// Quantisation, per 32 values x (each step rounded to f32 as written, so that any program following it gets the same
// bits):
//   q8_0: step = max|x| / 127, y = x * (1 / step), q = y to the nearest, halves away from zero; value q * f16(step)
//   q4_0: step = m / -8 with m the first x of the largest |x|, q = min(15, floor(x * (1 / step) + 8.5));
//         value (q - 8) * f16(step)
// A step that f16 rounds to zero stores zeros. A block that holds an infinity or a NaN, or whose step passes f16's
// range, is stored with a NaN scale: it reads back as NaN, where a clamped one would pass for data.
//
// Both directions are bound by memory: eight lanes take a block, four values each (a 16-byte load of f32 rows), K and
// V of the same place by the same lanes, so every thread has two loads in flight and a warp touches whole 128-byte
// lines on the f32 side and whole 32-byte sectors of the cache.
#include "kv.cuh"

namespace ocr {

constexpr int KV_THREADS = 256;

struct F4 {
    float x[4];
};
__device__ __forceinline__ F4 load4(const float* p) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    return {{v.x, v.y, v.z, v.w}};
}
__device__ __forceinline__ F4 load4(const __half* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    return {{a.x, a.y, b.x, b.y}};
}
__device__ __forceinline__ void store4(float* p, const F4& v) {
    *reinterpret_cast<float4*>(p) = make_float4(v.x[0], v.x[1], v.x[2], v.x[3]);
}
__device__ __forceinline__ uint2 half4(const F4& v) {
    const __half2 a = __floats2half2_rn(v.x[0], v.x[1]), b = __floats2half2_rn(v.x[2], v.x[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__half* p, const F4& v) { *reinterpret_cast<uint2*>(p) = half4(v); }

// Four values of a block by lane l (0 … 7) of its eight; all 32 lanes of the warp call it.
template <int TYPE>
__device__ __forceinline__ void quantise4(const F4& v, int lane, uint8_t* q, __half* scale, bool write) {
    const int l = lane & 7;
    const unsigned mine = 0xffu << (lane & 24);
    float big = 0.0f, m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = fabsf(v.x[i]);
        bad |= !(a <= 3.4028234e38f);
        if (a > big) big = a, m = v.x[i];
    }
    float top = big;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
    bad = (__ballot_sync(FULL, bad) & mine) != 0;
    float step;
    if (TYPE == KV_Q8_0) {
        step = __fdiv_rn(top, 127.0f);
    } else {  // the first of the largest: the lowest lane that holds one, and in it the first
        const unsigned has = __ballot_sync(FULL, big == top) & mine;
        step = __shfl_sync(FULL, m, has ? __ffs(has) - 1 : lane) * -0.125f;
    }
    const __half h = __float2half_rn(step);
    const float hs = fabsf(__half2float(h));
    bad |= !(hs <= 65504.0f);
    const bool zero = bad || hs == 0.0f;
    const float inv = zero ? 0.0f : __fdiv_rn(1.0f, step);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = zero ? 0.0f : __fmul_rn(v.x[i], inv);
        const uint32_t n = TYPE == KV_Q8_0 ? (uint32_t)__float2int_rz(roundf(y)) & 0xffu
                                           : (uint32_t)min(15, __float2int_rz(__fadd_rn(y, 8.5f)));
        w |= n << (8 * i);
    }
    if (TYPE == KV_Q4_0) {  // values j (low nibble) and j + 16 share a byte: lanes l and l + 4
        const uint32_t up = __shfl_xor_sync(FULL, w, 4);
        if (write && l < 4) *reinterpret_cast<uint32_t*>(q + 4 * l) = w | (up << 4);
    } else if (write) {
        *reinterpret_cast<uint32_t*>(q + 4 * l) = w;
    }
    if (write && l == 0) *scale = bad ? __ushort_as_half(0x7e00) : h;
}

// the four values of lane l of a block
template <int TYPE>
__device__ __forceinline__ F4 values4(const uint8_t* q, __half scale, int l) {
    F4 v;
    const float d = __half2float(scale);
    if (TYPE == KV_Q8_0) {
        i8x4_to_f32(*reinterpret_cast<const uint32_t*>(q + 4 * l), v.x);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(q + 4 * (l & 3)) >> (l & 4);
#pragma unroll
        for (int i = 0; i < 4; i++) v.x[i] = (float)((w >> (8 * i)) & 15u) - 8.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v.x[i] *= d;
    return v;
}

template <int TYPE, bool WRITE, class T>
__global__ void __launch_bounds__(KV_THREADS) k_kv_move(KvMoveArgs a) {
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    const int lane = threadIdx.x & 31, l = lane & 7;
    const int nb = c.d / KV_BLOCK;
    // the block of this thread's eight lanes, in the order [slot][row][head][block]
    const long unit = ((long)blockIdx.x * KV_THREADS + threadIdx.x) >> 3;
    const long per_slot = (long)a.r.T * c.n_kv * nb;
    const int b = (int)(unit / per_slot);
    bool live = b < c.n_slot;
    int t = 0, h = 0, blk = 0;
    size_t at = 0;
    if (live) {
        const int u = (int)(unit - b * per_slot);
        blk = u % nb;
        h = (u / nb) % c.n_kv;
        t = u / (nb * c.n_kv);
        const bool inside = t < a.r.rows(c, b, a.err);
        if (!WRITE && !inside) {  // a row that is not in use reads as zeros
            const F4 z = {};
            store4(static_cast<T*>(a.k) + b * a.k_slot + t * a.k_row + h * a.k_head + blk * KV_BLOCK + 4 * l, z);
            store4(static_cast<T*>(a.v) + b * a.v_slot + t * a.v_row + h * a.v_head + blk * KV_BLOCK + 4 * l, z);
        }
        live = inside;
        if (live) at = kv_index(c, b, h, kv_row(c, a.r.pos[b] + t));
    }
    T* kp = static_cast<T*>(a.k) + b * a.k_slot + t * a.k_row + h * a.k_head + blk * KV_BLOCK + 4 * l;
    T* vp = static_cast<T*>(a.v) + b * a.v_slot + t * a.v_row + h * a.v_head + blk * KV_BLOCK + 4 * l;
    const size_t qo = at * kv_row_bytes(TYPE, c.d) + (size_t)blk * kv_row_bytes(TYPE, KV_BLOCK), so = at * nb + blk;
    if (TYPE == KV_F16) {
        if (!live) return;
        __half* kc = reinterpret_cast<__half*>(c.k + qo) + 4 * l;
        __half* vc = reinterpret_cast<__half*>(c.v + qo) + 4 * l;
        if (WRITE) {
            const F4 x = load4(kp), y = load4(vp);
            store4(kc, x);
            store4(vc, y);
        } else {
            const F4 x = load4(kc), y = load4(vc);
            store4(kp, x);
            store4(vp, y);
        }
    } else if (WRITE) {  // (every lane takes part in the block's shuffles)
        F4 x = {}, y = {};
        if (live) x = load4(kp), y = load4(vp);
        quantise4<TYPE>(x, lane, c.k + qo, c.ks + so, live);
        quantise4<TYPE>(y, lane, c.v + qo, c.vs + so, live);
    } else if (live) {
        const F4 x = values4<TYPE>(c.k + qo, c.ks[so], l), y = values4<TYPE>(c.v + qo, c.vs[so], l);
        store4(kp, x);
        store4(vp, y);
    }
}

template <int TYPE, bool WRITE>
static cudaError_t launch_move(cudaStream_t st, const KvMoveArgs& a, bool pdl) {
    const long threads = (long)a.c.n_slot * a.r.T * a.c.n_kv * (a.c.d / KV_BLOCK) * 8;
    const dim3 grid((unsigned)((threads + KV_THREADS - 1) / KV_THREADS));
    return a.half ? kv_launch(k_kv_move<TYPE, WRITE, __half>, grid, KV_THREADS, 0, st, pdl, a)
                  : kv_launch(k_kv_move<TYPE, WRITE, float>, grid, KV_THREADS, 0, st, pdl, a);
}
template <bool WRITE>
static cudaError_t launch_move_type(cudaStream_t st, const KvMoveArgs& a, bool pdl) {
    switch (a.c.type) {
        case KV_F16: return launch_move<KV_F16, WRITE>(st, a, pdl);
        case KV_Q8_0: return launch_move<KV_Q8_0, WRITE>(st, a, pdl);
        default: return launch_move<KV_Q4_0, WRITE>(st, a, pdl);
    }
}
cudaError_t launch_kv_write(cudaStream_t st, const KvMoveArgs& a, bool pdl) { return launch_move_type<true>(st, a, pdl); }
cudaError_t launch_kv_read(cudaStream_t st, const KvMoveArgs& a, bool pdl) { return launch_move_type<false>(st, a, pdl); }

// ---- the accepted drafts' rows -----------------------------------------------------------------------------------------
// One CTA per (slot, kv head, layer): row pos + path[i] moves to row pos + i. path rises strictly and path[i] >= i, so
// a destination may be a later source: every row is in shared memory before the first is written. Latency-bound: one
// round trip to memory, at most KV_TREE_MAX rows.
__global__ void __launch_bounds__(128) k_kv_keep(const __grid_constant__ KvKeepArgs a) {
    extern __shared__ uint4 held[];  // K rows, V rows, K scales, V scales
    __shared__ int src[KV_TREE_MAX], dst[KV_TREE_MAX];
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const auto& L = a.layer[blockIdx.z];
    const int pos = a.pos[b], n = a.n[b];
    if (pos < 0 || n <= 0) return;
    bool ok = n <= a.T && (c.ring ? (long)pos + a.T <= 0x7fffffffL : (long)pos + a.T <= (long)c.n_rows);
    if (!ok) {
        if (tid == 0) dev_error(a.err, DEV_BAD_POS);
        return;
    }
    bool bad = false;
    if (tid < n) {
        const int p = a.path[(size_t)b * a.T + tid];
        bad = p < tid || p >= a.T || (tid > 0 && a.path[(size_t)b * a.T + tid - 1] >= p);
        src[tid] = kv_row(c, pos + (bad ? tid : p));
        dst[tid] = kv_row(c, pos + tid);
    }
    if (__syncthreads_or(bad)) {
        if (tid == 0) dev_error(a.err, DEV_BAD_INDEX);
        return;
    }
    const int rb = kv_row_bytes(c.type, c.d), pieces = rb / 16;
    const int nb = c.type == KV_F16 ? 0 : c.d / KV_BLOCK;
    __half* hs = reinterpret_cast<__half*>(held + 2 * KV_TREE_MAX * pieces);
    const size_t base = kv_index(c, b, h, 0);
    for (int e = tid; e < n * pieces; e += 128) {
        const size_t o = (base + src[e / pieces]) * rb + (size_t)(e % pieces) * 16;
        held[e] = *reinterpret_cast<const uint4*>(L.k + o);
        held[KV_TREE_MAX * pieces + e] = *reinterpret_cast<const uint4*>(L.v + o);
    }
    for (int e = tid; e < n * nb; e += 128) {
        const size_t o = (base + src[e / nb]) * nb + e % nb;
        hs[e] = L.ks[o];
        hs[KV_TREE_MAX * nb + e] = L.vs[o];
    }
    __syncthreads();
    for (int e = tid; e < n * pieces; e += 128) {
        const size_t o = (base + dst[e / pieces]) * rb + (size_t)(e % pieces) * 16;
        *reinterpret_cast<uint4*>(L.k + o) = held[e];
        *reinterpret_cast<uint4*>(L.v + o) = held[KV_TREE_MAX * pieces + e];
    }
    for (int e = tid; e < n * nb; e += 128) {
        const size_t o = (base + dst[e / nb]) * nb + e % nb;
        L.ks[o] = hs[e];
        L.vs[o] = hs[KV_TREE_MAX * nb + e];
    }
}

cudaError_t launch_kv_keep(cudaStream_t st, const KvKeepArgs& a, bool pdl) {
    const size_t smem = 2 * KV_TREE_MAX * ((size_t)kv_row_bytes(a.c.type, a.c.d) + a.c.d / KV_BLOCK * 2);
    return kv_launch(k_kv_keep, dim3(a.c.n_kv, a.c.n_slot, a.n_layer), 128, smem, st, pdl, a);
}

}  // namespace ocr
