// kv_tile.cuh — key tiles of a KV cache streamed through shared memory by the attentions of few rows (k_kv_attn.cu,
// k_kv_attn_one.cu): a tile's layout, and a team of warps' ring of asynchronous copies.
#pragma once

#include "kv_attn.cuh"

namespace ocr {

constexpr int KA_RING = 17408;       // a warp's share of the rings: two q8_0 tiles of 32 keys

template <int TYPE, int D>
struct KaTile {
    static constexpr int ROW = kv_row_bytes(TYPE, D);
    static constexpr int NB = TYPE == KV_F16 ? 0 : D / KV_BLOCK;
    static constexpr int KEYS = TYPE == KV_F16 ? 2048 / D : TYPE == KV_Q8_0 ? 4096 / D : D == 128 ? 32 : 64;
    static constexpr int K_BYTES = KEYS * ROW, S_BYTES = KEYS * NB * 2;
    static constexpr int STAGE = 2 * (K_BYTES + S_BYTES);  // K, V, K scales, V scales
    static constexpr int STAGES = KA_RING / STAGE;         // per warp
    // the byte offset of 16-byte piece c of key i: permuted so that the eight (K) or four (V) keys that a warp reads at
    // once lie in different banks
    __device__ static __forceinline__ int off(int i, int c, bool v) {
        if (TYPE == KV_F16) return i * ROW + ((c ^ (i & 7)) << 4);
        if (TYPE == KV_Q8_0 && D == 128)
            return i * ROW + ((c ^ ((v ? (i >> 2) & 3 : (i & 1) | ((i >> 1) & 2)) << 1)) << 4);
        if (TYPE == KV_Q8_0) return (i ^ ((i >> 3) & 1)) * ROW + ((c ^ (((i >> 2) & 1) << 1)) << 4);
        if (D == 128) return i * ROW + ((c ^ ((i >> 2) & 3)) << 4);
        return (i ^ (((i >> 3) & 1) << 1)) * ROW + ((c ^ ((i >> 2) & 1)) << 4);
    }
};

// a key's NB scales
template <int NB>
__device__ __forceinline__ void load_scales(__half2* d, const uint8_t* scales, int key) {
    if constexpr (NB == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(scales + key * 8);
        d[0] = *reinterpret_cast<const __half2*>(&x.x), d[1] = *reinterpret_cast<const __half2*>(&x.y);
    } else {
        d[0] = *reinterpret_cast<const __half2*>(scales + key * 4);
    }
}
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
    const int n = live ? N : 0;  // the rest is filled with zeros
    if (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Short pairs are taken whole: a pair costs the time of some KA_PIECE tiles beside its own (queries, the teams joined), as
// much again where it is cut (parts written, counted, joined). 32 slots, 8 kv heads, a window of 1024 in q4_0 (256 pairs
// of 33 tiles): 25 us whole, 32 cut.
constexpr int KA_PIECE = 14;
struct KaLine {
    int prefix[KA_LINE + 1], pos[KA_LINE], m[KA_LINE];  // of the slots: tiles before, position, rows in use
    int wsum[32], longest;                              // the most tiles of a pair
};
// The copies of a team's tiles (WR warps share a ring; team i of TEAMS takes tiles begin + i, begin + i + TEAMS, …).
template <int TYPE, int D, int WR, int TEAMS>
struct KaStream {
    using KT = KaTile<TYPE, D>;
    static constexpr int STAGES = KT::STAGES * WR, KEYS = KT::KEYS, NB = KT::NB;
    static constexpr int PIECES = KT::ROW / 16, KEYS_PER = 32 * WR / PIECES;  // 16-byte pieces of a key; keys of one round
    const KvAttnArgs& a;
    const KaLine& line;
    KvCursor at;
    KvSpan s;
    uint32_t ring;
    int next, end, count = 0, tl, lkey, lpiece;  // the next tile to copy, the copies so far
    __device__ __forceinline__ KaStream(const KvAttnArgs& a_, const KaLine& line_, int begin, int end_, int team, int tl_,
                                        const uint8_t* ring_)
        : a(a_), line(line_), ring(smem_u32(ring_)), next(begin + team), end(end_), tl(tl_), lkey(tl_ / PIECES),
          lpiece(tl_ % PIECES) {
        go(begin);
    }
    __device__ __forceinline__ void go(int tile) {
        at.at(tile, line.prefix, a.c.n_slot, a.c.n_kv);
        s.set(a, line.pos[at.b], line.m[at.b], 0, a.r.T);
    }
    __device__ __forceinline__ void load() {  // the next tile, if there is one; a group of copies either way
        if (next < end) {
            const KvView& c = a.c;
            if (next >= at.first + at.tiles) go(next);
            const uint32_t dst = ring + count % STAGES * KT::STAGE;
            const int v0 = (next - at.first) * KEYS, v1 = v0 + KEYS - 1;
            const size_t base = kv_index(c, at.b, at.h, 0);
            const int r0 = kv_row(c, s.position(v0));
            // a tile whose rows lie one after another: one base, constant steps
            if (v1 < s.nv && (v0 >= s.ns || v1 < s.ns) && kv_row(c, s.position(v1)) - r0 == KEYS - 1) {
                const size_t row = base + r0;
                const uint8_t *kp = c.k + (row + lkey) * KT::ROW + lpiece * 16, *vp = c.v + (row + lkey) * KT::ROW + lpiece * 16;
#pragma unroll
                for (int e = 0; e < KEYS / KEYS_PER; e++) {
                    const int i = lkey + e * KEYS_PER;
                    cp_async<16>(dst + KT::off(i, lpiece, false), kp + e * KEYS_PER * KT::ROW, true);
                    cp_async<16>(dst + KT::K_BYTES + KT::off(i, lpiece, true), vp + e * KEYS_PER * KT::ROW, true);
                }
                if constexpr (NB > 0) {
                    const __half *ks = c.ks + (row + tl) * NB, *vs = c.vs + (row + tl) * NB;
#pragma unroll
                    for (int i = 0; i < KEYS; i += 32 * WR) {
                        if (i + tl >= KEYS) break;
                        cp_async<NB * 2>(dst + 2 * KT::K_BYTES + (i + tl) * NB * 2, ks + i * NB, true);
                        cp_async<NB * 2>(dst + 2 * KT::K_BYTES + KT::S_BYTES + (i + tl) * NB * 2, vs + i * NB, true);
                    }
                }
            } else {
#pragma unroll 1
                for (int i = lkey; i < KEYS; i += KEYS_PER) {
                    const bool live = v0 + i < s.nv;
                    const size_t row = base + (live ? kv_row(c, s.position(v0 + i)) : 0);
                    cp_async<16>(dst + KT::off(i, lpiece, false), c.k + row * KT::ROW + lpiece * 16, live);
                    cp_async<16>(dst + KT::K_BYTES + KT::off(i, lpiece, true), c.v + row * KT::ROW + lpiece * 16, live);
                }
                if constexpr (NB > 0) {
#pragma unroll 1
                    for (int i = tl; i < KEYS; i += 32 * WR) {
                        const bool live = v0 + i < s.nv;
                        const size_t row = base + (live ? kv_row(c, s.position(v0 + i)) : 0);
                        cp_async<NB * 2>(dst + 2 * KT::K_BYTES + i * NB * 2, c.ks + row * NB, live);
                        cp_async<NB * 2>(dst + 2 * KT::K_BYTES + KT::S_BYTES + i * NB * 2, c.vs + row * NB, live);
                    }
                }
            }
            next += TEAMS;
            count++;
        }
        cp_commit();
    }
};

// The line of tiles of all (slot, kv head) pairs; rows that are not in use are set to zeros on the way. → the line's
// length
template <int KEYS, int D, class T, int THREADS>
__device__ __forceinline__ int kv_line_sums(const KvAttnArgs& a, KaLine& line) {
    static_assert(THREADS >= KA_LINE, "a thread per slot");
    const KvView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    KvSpan span;
    span.nv = 0;
    bool idle_rows = false;
    if (tid < c.n_slot) {
        span.set(a, tid, 0, a.r.T);
        idle_rows = span.m < a.r.T;
        line.pos[tid] = span.pos, line.m[tid] = span.m;
    }
    if (tid == 0) line.longest = 0;
    const int tiles = (span.nv + KEYS - 1) / KEYS;
    int x = tiles * c.n_kv;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) line.wsum[warp] = x;
    idle_rows = __syncthreads_or(idle_rows);
    const int most = __reduce_max_sync(FULL, tiles);
    if (lane == 0 && most) atomicMax(&line.longest, most);
    int total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) x += line.wsum[w];
        total += line.wsum[w];
    }
    if (tid < c.n_slot) line.prefix[tid + 1] = x;
    if (tid == 0) line.prefix[0] = 0;
    __syncthreads();
    if (idle_rows) {
        const long n = (long)c.n_slot * a.r.T * a.n_head;
        for (long i = (long)blockIdx.x * (THREADS / 32) + warp; i < n; i += (long)gridDim.x * (THREADS / 32)) {
            const int h = (int)(i % a.n_head), r = (int)(i / a.n_head % a.r.T), b = (int)(i / a.n_head / a.r.T);
            if (r < a.r.rows(c, b, nullptr)) continue;
            T* o = static_cast<T*>(a.out) + b * a.o_slot + r * a.o_row + h * a.o_head;
            for (int d = lane; d < D; d += 32) o[d] = (T)0.0f;
        }
    }
    return total;
}

}  // namespace ocr
