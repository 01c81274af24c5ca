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
// lines on the f32 side and whole 32-byte sectors of the cache. 32 slots, 2214 rows, 8 heads of 128 in q8_0 (580 MB of
// rows, 154 MB of cache): written in 172 us (4.3 TB/s), read back in 144 (5.1).
#include "kv.cuh"

namespace ocr {

constexpr int KV_THREADS = 256;
constexpr int KV_ROWS = 2;  // rows of a thread: K and V of each in flight together

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

template <int TYPE, int D, bool WRITE, class T>
__global__ void __launch_bounds__(KV_THREADS) k_kv_move(const __grid_constant__ KvMoveArgs a, unsigned rows_step) {
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    constexpr int NB = D / KV_BLOCK;
    const int lane = threadIdx.x & 31, l = lane & 7;
    // this thread's eight lanes take block blk of head h, of slot blockIdx.y's rows t, t + rows_step (one division here;
    // the rows of a slot in one launch are few enough for 32 bits)
    const unsigned unit = (blockIdx.x * KV_THREADS + threadIdx.x) >> 3;
    const unsigned head = unit / NB, t0 = head / (unsigned)c.n_kv;
    const int blk = unit % NB, h = (int)(head - t0 * c.n_kv), b = blockIdx.y;
    const int n = a.r.rows(c, b, a.err), pos = a.r.pos[b];
    const size_t base = kv_index(c, b, h, 0);
    const long ko = b * a.k_slot + h * a.k_head + blk * KV_BLOCK + 4 * l, vo = b * a.v_slot + h * a.v_head + blk * KV_BLOCK + 4 * l;
    constexpr int RB = kv_row_bytes(TYPE, D), BB = kv_row_bytes(TYPE, KV_BLOCK);
    F4 x[KV_ROWS], y[KV_ROWS];
    size_t at[KV_ROWS];
    bool live[KV_ROWS];
#pragma unroll
    for (int i = 0; i < KV_ROWS; i++) {
        const unsigned t = t0 + i * rows_step;
        live[i] = t < (unsigned)n && (i > 0 || t < rows_step);  // (past the first share: the next thread's)
        at[i] = base + (live[i] ? kv_row(c, pos + (int)t) : 0);
        x[i] = y[i] = F4{};
        if (WRITE) {
            if (live[i]) x[i] = load4(static_cast<const T*>(a.k) + ko + t * a.k_row), y[i] = load4(static_cast<const T*>(a.v) + vo + t * a.v_row);
        } else if (live[i]) {
            const uint8_t *kq = c.k + at[i] * RB + blk * BB, *vq = c.v + at[i] * RB + blk * BB;
            if constexpr (TYPE == KV_F16) {
                x[i] = load4(reinterpret_cast<const __half*>(kq) + 4 * l), y[i] = load4(reinterpret_cast<const __half*>(vq) + 4 * l);
            } else {
                x[i] = values4<TYPE>(kq, c.ks[at[i] * NB + blk], l), y[i] = values4<TYPE>(vq, c.vs[at[i] * NB + blk], l);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < KV_ROWS; i++) {
        const unsigned t = t0 + i * rows_step;
        if (!WRITE) {  // (a row that is not in use reads as zeros)
            if (t >= (unsigned)a.r.T || (i == 0 && t >= rows_step)) continue;
            store4(static_cast<T*>(a.k) + ko + t * a.k_row, x[i]);
            store4(static_cast<T*>(a.v) + vo + t * a.v_row, y[i]);
        } else if constexpr (TYPE == KV_F16) {
            if (!live[i]) continue;
            store4(reinterpret_cast<__half*>(c.k + at[i] * RB + blk * BB) + 4 * l, x[i]);
            store4(reinterpret_cast<__half*>(c.v + at[i] * RB + blk * BB) + 4 * l, y[i]);
        } else {  // (every lane takes part in the block's shuffles)
            quantise4<TYPE>(x[i], lane, c.k + at[i] * RB + blk * BB, c.ks + at[i] * NB + blk, live[i]);
            quantise4<TYPE>(y[i], lane, c.v + at[i] * RB + blk * BB, c.vs + at[i] * NB + blk, live[i]);
        }
    }
}

template <int TYPE, int D, bool WRITE>
static cudaError_t launch_move(cudaStream_t st, const KvMoveArgs& a, bool pdl) {
    const unsigned step = (unsigned)(a.r.T + KV_ROWS - 1) / KV_ROWS;
    const long threads = (long)step * a.c.n_kv * (D / KV_BLOCK) * 8;
    const dim3 grid((unsigned)((threads + KV_THREADS - 1) / KV_THREADS), a.c.n_slot);
    return a.half ? kv_launch(k_kv_move<TYPE, D, WRITE, __half>, grid, KV_THREADS, 0, st, pdl, a, step)
                  : kv_launch(k_kv_move<TYPE, D, WRITE, float>, grid, KV_THREADS, 0, st, pdl, a, step);
}
template <bool WRITE>
static cudaError_t launch_move_type(cudaStream_t st, const KvMoveArgs& a, bool pdl) {
    const bool wide = a.c.d == 128;
    switch (a.c.type) {
        case KV_F16: return wide ? launch_move<KV_F16, 128, WRITE>(st, a, pdl) : launch_move<KV_F16, 64, WRITE>(st, a, pdl);
        case KV_Q8_0: return wide ? launch_move<KV_Q8_0, 128, WRITE>(st, a, pdl) : launch_move<KV_Q8_0, 64, WRITE>(st, a, pdl);
        default: return wide ? launch_move<KV_Q4_0, 128, WRITE>(st, a, pdl) : launch_move<KV_Q4_0, 64, WRITE>(st, a, pdl);
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
    if (n > a.T) {
        if (tid == 0) dev_error(a.err, DEV_BAD_POS);
        return;
    }
    // (of the step's rows only those that the path names have to lie in the cache: a slot may have used fewer than T)
    bool bad = false, outside = false;
    if (tid < n) {
        const int p = a.path[(size_t)b * a.T + tid];
        bad = p < tid || p >= a.T || (tid > 0 && a.path[(size_t)b * a.T + tid - 1] >= p);
        outside = !bad && (long)pos + p >= (c.ring ? 0x7fffffffL : (long)c.n_rows);
        if (!bad && !outside) {
            src[tid] = kv_row(c, pos + p);
            dst[tid] = kv_row(c, pos + tid);
        }
    }
    bad = __syncthreads_or(bad);
    outside = __syncthreads_or(outside);
    if (bad || outside) {
        if (tid == 0) dev_error(a.err, bad ? DEV_BAD_INDEX : DEV_BAD_POS);
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
