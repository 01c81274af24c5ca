// k_kv_attn.cu — attention of a few rows per kv head (a decode step, a small tree of drafts) over a KV cache (kv.cuh).
//
// out[t] = sum_p softmax_p(scale q_t . k_p) v_p over the visible positions p: p <= pos + t, and with a window also
// p > pos + t - window or p < sinks. Drafts (a parent for each row): row t stands at position pos + depth(t) and sees
// the committed positions and, of the drafts, its ancestors and itself. A row that sees nothing gives zeros.
//
// Bound: memory — each visible row of the cache is read once for all rows of the call. The work is cut evenly: the key
// tiles of all (slot, kv head) pairs form one line, CTA c of C takes the c-th part of it, its warps take the tiles in
// turn, whatever the lengths. A pair that lies in several CTAs is joined by the last of them to arrive (a ticket; the
// parts are added in the order of the CTAs, so the result does not depend on who is last). The warps stand in teams, one
// warp to eight of the rows; a team streams its tiles through a ring of its own with asynchronous copies (a named barrier
// where it has two or four warps) and meets the others only where a pair is joined; the ring runs on into the next pair
// meanwhile.
// Measured: 32 slots of some 3200 keys, 8 drafts each (16 rows to a kv head), q8_0: 140 us, 1.6 TB/s of cache; bound by
// instruction issue (the quants' way to f16 for each 8 columns) and by the pairs' fixed part. One slot of 2319 keys, 16
// drafts: 46 us, latency — a part of a few tiles, its join over the pair's CTAs.
//
// Products: warp-level tensor-core products m16n8k16 (f16 in, f32 out) with the keys as the 16 rows and up to eight
// (row, query head) pairs as the columns: S = K Q^T, then O = V^T P with the dims as the rows. A decode step has no use
// for the 128-row tcgen05 shapes, and the operands here come out of registers, where the quants become f16 — no pass
// through shared memory. Exactness: q8_0 and q4_0 quants are integers and exact in f16; a key's block scale multiplies
// the block's f32 partial score, a value's block scale goes into P (one P per block of 32 dims). f32 queries, and P,
// are split into f16 hi + lo (22 bits); f16 queries are exact, and P (times the scale) is rounded to f16 once, like the
// output. A row's query is scaled by a power of two so that its lo part does not fall below f16's range, P likewise by the tile's largest
// scale.
#include "kv_tile.cuh"

namespace ocr {

// (row, query head) pairs of a kv head up to which this kernel runs. In this kernel and in k_kv_attn_tc.cu: 16 pairs (a step of 32
// slots, 8 drafts, q8_0) 148 and 243 us; 32 pairs, one slot (a step of 16 drafts) 45 and 51; 32 pairs, 32 slots x 16 rows, 199 and
// 225 over q8_0, 175 and 195 over f16. More would need more than four warps to a team.
constexpr int KA_ROWS = 32;
constexpr int KA_WARPS = 12;
constexpr int KA_THREADS = KA_WARPS * 32;

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr));
}
template <int TYPE, int D, int WR, bool PACK, class T>
__global__ void __launch_bounds__(KA_THREADS, 1) k_kv_attn(const __grid_constant__ KvAttnArgs a) {
    using KT = KaTile<TYPE, D>;
    constexpr bool LO = sizeof(T) == 4 && !PACK;  // the lo halves of q and P in products of their own
    constexpr int TEAMS = KA_WARPS / WR;         // WR warps share a ring, eight rows each
    constexpr int STAGES = KaStream<TYPE, D, WR, TEAMS>::STAGES;
    constexpr int KEYS = KT::KEYS, MT = KEYS / 16, NB = KT::NB;
    constexpr int ROWS = PACK ? 4 : 8;           // of a warp: PACK has four in columns 0 … 3, their lo halves in 4 … 7
    constexpr int KSTEPS = D / 16, DT = D / 16;  // 16-dim steps of S, 16-dim tiles of O
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ KaLine line;
    __shared__ int s_parent[KV_TREE_MAX], s_depth[KV_TREE_MAX];
    __shared__ KvSight s_sight[8 * WR];
    __shared__ float s_ml[4][16];
    __shared__ int s_last;
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int team = warp / WR, wr = warp % WR, tl = tid - team * WR * 32;
    const int G = a.n_head / c.n_kv;

    const int total = kv_line_sums<KEYS, D, T, KA_THREADS>(a, line);
    // a short line takes fewer CTAs, and fewer parts to join
    const int share = kv_least_share(total, c.n_slot * c.n_kv, TEAMS), n_cta = min((int)gridDim.x, (total + share - 1) / share);
    const int cta = blockIdx.x;
    KvLine cut;
    cut.cut(total, n_cta);
    int begin, end;
    kv_share(cut, cta, line.prefix, c.n_slot, c.n_kv, total, line.longest, (int)gridDim.x, KA_PIECE, KA_PIECE, begin, end);
    if (begin >= end) return;

    uint8_t* ring = smem + team * WR * KA_RING;
    float* joined = reinterpret_cast<float*>(smem + KA_WARPS * KA_RING);  // [4 warps][D / 4 registers][32 lanes]

    // ---- the copies of a tile, by the team's threads ----
    KaStream<TYPE, D, WR, TEAMS> stream(a, line, begin, end, team, tl, ring);
    auto load = [&]() { stream.load(); };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) load();

    int done = 0;  // tiles computed by the team
    int ct = begin + team;
    for (int seg = begin; seg < end;) {
        KvCursor cc;
        KvSpan sp;
        cc.at(seg, line.prefix, c.n_slot, c.n_kv);
        sp.set(a, line.pos[cc.b], line.m[cc.b], 0, a.r.T);
        const int seg_end = min(end, cc.first + cc.tiles);
        const int rows = sp.m * G;
        const bool many = a.r.T > 1 || a.parent;  // (else every row sees the whole span)
        // ---- what each row sees ----
        if (many) {
            if (a.parent) {
                if (tid < sp.m) s_parent[tid] = a.parent[(size_t)cc.b * a.r.T + tid];
                __syncthreads();
                if (tid < sp.m) s_depth[tid] = kv_depth(tid, s_parent, a.err);
                __syncthreads();
            }
            if (tid < 8 * WR) {
                const int row = min(tid / G, sp.m - 1);
                if (a.parent)
                    kv_draft(c, sp, row, s_parent, s_depth, s_sight[tid]);
                else
                    s_sight[tid].rows(c, sp, sp.pos + row, sp.pos + row);
            }
            __syncthreads();
        }
        // ---- this warp's queries, as the products' B operand: column g is row 8 wr + g ----
        uint32_t qh[KSTEPS][2], ql[LO ? KSTEPS : 1][2];
        float sfac[2];
        {
            const int r = ROWS * wr + (PACK ? g & 3 : g);
            const bool live = r < rows;
            const T* qp = static_cast<const T*>(a.q) + cc.b * a.q_slot + (r / G) * a.q_row + (cc.h * G + r % G) * a.q_head;
            float x[D / 4];  // the lane's dims: of step s, k = 2t, 2t + 1, 2t + 8, 2t + 9 at x[4 s …]
#pragma unroll
            for (int s = 0; s < KSTEPS; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    int d;
                    if (TYPE == KV_F16)
                        d = 16 * s + 2 * t + (i & 1) + 8 * (i >> 1);
                    else if (TYPE == KV_Q8_0)
                        d = 32 * (s >> 1) + 8 * t + 4 * (s & 1) + i;
                    else  // bytes 4t … 4t + 3 of the block: pairs (0, 2), (1, 3)
                        d = 32 * (s >> 1) + 16 * (s & 1) + 4 * t + ((i & 1) << 1) + (i >> 1);
                    x[4 * s + i] = live ? (float)qp[d] : 0.0f;
                }
            float f = a.scale * LOG2E;
            if constexpr (sizeof(T) == 4) {
                // the row times a power of two that brings its largest to 2^10 … 2^11 (an infinity or a NaN: 1)
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 4; i++) big = fmaxf(big, fabsf(x[i]));
                big = fmaxf(big, __shfl_xor_sync(FULL, big, 1));
                big = fmaxf(big, __shfl_xor_sync(FULL, big, 2));
                const int e = big > 0.0f && big <= 3.4028234e38f ? min(100, 137 - (int)(__float_as_uint(big) >> 23)) : 0;
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                f *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int i = 0; i < D / 4; i++) x[i] *= up;
            }
#pragma unroll
            for (int s = 0; s < KSTEPS; s++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    qh[s][i] = sizeof(T) == 4 && TYPE == KV_F16 ? pack2_below(x[4 * s + 2 * i], x[4 * s + 2 * i + 1])
                                                                : pack2(x[4 * s + 2 * i], x[4 * s + 2 * i + 1]);
                    if constexpr (PACK) {
                        const uint32_t lo = rest2(x[4 * s + 2 * i], x[4 * s + 2 * i + 1], qh[s][i]);
                        if (g >= 4) qh[s][i] = lo;
                    }
                    if constexpr (LO) ql[s][i] = rest2(x[4 * s + 2 * i], x[4 * s + 2 * i + 1], qh[s][i]);
                }
            // column 2t and 2t + 1's factor (held by the lanes of g = 2t, 2t + 1)
            sfac[0] = __shfl_sync(FULL, f, 8 * t);
            sfac[1] = __shfl_sync(FULL, f, 8 * t + 4);
        }
        float o[DT][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        // ---- a tile ----
        auto compute = [&](int tile, const uint8_t* st, auto edge_) {
            constexpr bool EDGE = decltype(edge_)::value;
            const uint8_t *kt = st, *vt = st + KT::K_BYTES;
            [[maybe_unused]] const uint8_t *kst = st + 2 * KT::K_BYTES, *vst = kst + KT::S_BYTES;
            const int v0 = (tile - cc.first) * KEYS;
            float p[MT][4];
            // S: rows g and g + 8 of 16 keys are keys kA and kB, columns 2t and 2t + 1. f16: keys g and g + 8; quants:
            // the order in which one lane's four keys of V's transposition are 4t … 4t + 3
            auto key = [&](int i, int up) {
                return 16 * i + (TYPE == KV_F16 ? g + 8 * up : 4 * (g >> 1) + (g & 1) + 2 * up);
            };
#pragma unroll
            for (int i = 0; i < MT; i++) {
                if constexpr (TYPE == KV_F16) {
                    float acc[4] = {};
#pragma unroll
                    for (int s = 0; s < KSTEPS; s++) {
                        uint32_t ka[4];
                        ldmatrix4<false>(ka, smem_u32(kt + KT::off(16 * i + (lane & 15), 2 * s + (lane >> 4), false)));
                        mma16816(acc, ka, qh[s][0], qh[s][1]);
                        if constexpr (LO) mma16816(acc, ka, ql[s][0], ql[s][1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) p[i][j] = acc[j];
                } else {
                    const int kA = key(i, 0), kB = key(i, 1);
#pragma unroll
                    for (int j = 0; j < 4; j++) p[i][j] = 0.0f;
                    __half2 dk[2][NB / 2];
                    load_scales<NB>(dk[0], kst, kA), load_scales<NB>(dk[1], kst, kB);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t ka[2][4];
                        if constexpr (TYPE == KV_Q8_0) {
                            const uint2 wA = *reinterpret_cast<const uint2*>(kt + KT::off(kA, 2 * b + (t >> 1), false) + (t & 1) * 8);
                            const uint2 wB = *reinterpret_cast<const uint2*>(kt + KT::off(kB, 2 * b + (t >> 1), false) + (t & 1) * 8);
#pragma unroll
                            for (int s = 0; s < 2; s++) {
                                const uint32_t A = (s ? wA.y : wA.x) ^ 0x80808080u, B = (s ? wB.y : wB.x) ^ 0x80808080u;
                                ka[s][0] = bytes_h2(A, 0x4140, H2_1152), ka[s][2] = bytes_h2(A, 0x4342, H2_1152);
                                ka[s][1] = bytes_h2(B, 0x4140, H2_1152), ka[s][3] = bytes_h2(B, 0x4342, H2_1152);
                            }
                        } else {
                            const uint32_t A = *reinterpret_cast<const uint32_t*>(kt + KT::off(kA, b, false) + t * 4);
                            const uint32_t B = *reinterpret_cast<const uint32_t*>(kt + KT::off(kB, b, false) + t * 4);
                            ka[0][0] = nibbles_h2<false>(A), ka[0][2] = nibbles_h2<false>(A >> 8);
                            ka[1][0] = nibbles_h2<true>(A), ka[1][2] = nibbles_h2<true>(A >> 8);
                            ka[0][1] = nibbles_h2<false>(B), ka[0][3] = nibbles_h2<false>(B >> 8);
                            ka[1][1] = nibbles_h2<true>(B), ka[1][3] = nibbles_h2<true>(B >> 8);
                        }
                        float acc[4] = {};
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            mma16816(acc, ka[s], qh[2 * b + s][0], qh[2 * b + s][1]);
                            if constexpr (LO) mma16816(acc, ka[s], ql[2 * b + s][0], ql[2 * b + s][1]);
                        }
                        const float dA = b & 1 ? __high2float(dk[0][b / 2]) : __low2float(dk[0][b / 2]);
                        const float dB = b & 1 ? __high2float(dk[1][b / 2]) : __low2float(dk[1][b / 2]);
                        p[i][0] = fmaf(acc[0], dA, p[i][0]), p[i][1] = fmaf(acc[1], dA, p[i][1]);
                        p[i][2] = fmaf(acc[2], dB, p[i][2]), p[i][3] = fmaf(acc[3], dB, p[i][3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (PACK) p[i][j] += __shfl_xor_sync(FULL, p[i][j], 2);  // hi and lo
                    p[i][j] *= sfac[j & 1];
                }
            }
            // ---- the mask ----
            uint32_t bad = 0;       // (f16) keys of the tile whose values are not all finite
            [[maybe_unused]] uint64_t col_seen = 0;  // those that column g's row sees
            if constexpr (EDGE) {
                if (TYPE == KV_F16 && many) {
                    // a value that some rows see and some do not must not reach the latter as 0 * inf: such rows of V
                    // are taken out of the product and given to those who see them as a NaN weight
                    for (int i = 0; i < KEYS; i++) {
                        bool b = false;
                        if (lane < KT::ROW / 16) {
                            const uint4 x = *reinterpret_cast<const uint4*>(vt + KT::off(i, lane, true));
                            auto inf = [](uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; };
                            b = inf(x.x) || inf(x.y) || inf(x.z) || inf(x.w);
                        }
                        if (__any_sync(FULL, b)) bad |= 1u << i;
                    }
                }
                auto sees = [&](int col, int v) {
                    const int left = sp.nv - v;
                    return many ? s_sight[ROWS * wr + (col & (ROWS - 1))].mask(v)
                                : left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
                };
                if constexpr (NB > 0)
#pragma unroll
                    for (int w = 0; w < (KEYS + 31) / 32; w++) col_seen |= (uint64_t)sees(g, v0 + 32 * w) << (32 * w);
                uint32_t mask[2][(KEYS + 31) / 32];  // the tile's keys that the lane's two rows see
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int w = 0; w < (KEYS + 31) / 32; w++) mask[j][w] = sees(2 * t + j, v0 + 32 * w);
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int kk = key(i, j >> 1);
                        const bool s = (mask[j & 1][i / 2] >> (kk & 31)) & 1;
                        if (TYPE == KV_F16 && s && ((bad >> kk) & 1)) p[i][j] = NAN;
                        if (!s) p[i][j] = -INFINITY;
                    }
            }
            // ---- the running maximum, the weights ----
            float alpha[2], ref[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = fmaxf(p[0][j], p[0][j + 2]);
#pragma unroll
                for (int i = 1; i < MT; i++) x = fmaxf(x, fmaxf(p[i][j], p[i][j + 2]));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 4));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 8));
                x = fmaxf(x, __shfl_xor_sync(FULL, x, 16));
                const float mn = fmaxf(m[j], x), safe = mn == -INFINITY ? 0.0f : mn;
                alpha[j] = ex2(m[j] - safe);
                ref[j] = safe - 8.0f;  // weights up to 2^8: the small ones stay further from f16's smallest
                m[j] = mn;
                l[j] *= alpha[j];
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[i][j] = ex2(p[i][j] - ref[j & 1]);
                    l[j & 1] += p[i][j];
                }
            // ---- O = O alpha + V^T P: P as the B operand has column g, keys 2t, 2t + 1, 2t + 8, 2t + 9 of 16 ----
            uint32_t ph[MT][2];
            [[maybe_unused]] uint32_t pl[MT][2];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t h = pack2(p[i][2 * j], p[i][2 * j + 1]);
                    if constexpr (sizeof(T) == 4 || TYPE != KV_F16) {  // (over quants the product with the scale is rounded)
                        const uint32_t r = rest2(p[i][2 * j], p[i][2 * j + 1], h);
                        if (PACK && TYPE == KV_F16) {
                            ph[i][j] = transpose8(t < 2 ? h : r);
                        } else {
                            ph[i][j] = transpose8(h);
                            pl[i][j] = transpose8(r);
                        }
                    } else {
                        ph[i][j] = transpose8(h);
                    }
                }
            if constexpr (TYPE == KV_F16) {
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    float acc[4] = {};
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        uint32_t va[4];
                        ldmatrix4<true>(va, smem_u32(vt + KT::off(16 * i + (lane & 7) + ((lane >> 4) << 3),
                                                                 2 * d + ((lane >> 3) & 1), true)));
                        if (EDGE && bad) {  // keys 2t, 2t + 1 (registers 0, 1) and 2t + 8, 2t + 9 (2, 3)
                            const uint32_t z = bad >> (16 * i + 2 * t);
                            const uint32_t k0 = (z & 1 ? 0u : 0xffffu) | (z & 2 ? 0u : 0xffff0000u);
                            const uint32_t k1 = (z & 0x100 ? 0u : 0xffffu) | (z & 0x200 ? 0u : 0xffff0000u);
                            va[0] &= k0, va[1] &= k0, va[2] &= k1, va[3] &= k1;
                        }
                        mma16816(acc, va, ph[i][0], ph[i][1]);
                        if constexpr (LO) mma16816(acc, va, pl[i][0], pl[i][1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) o[d][j] = fmaf(o[d][j], alpha[j & 1], acc[j]);
                }
            } else {
                // the weights again in 32 bits, the scales of the lane's four keys of each 16 (4t … 4t + 3), and the
                // tile's largest of each block
                float w[MT][4];
                __half2 dv[MT][4][NB / 2], top[NB / 2];
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&ph[i][u]));
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&pl[i][u]));
                        w[i][2 * u] = h.x + r.x, w[i][2 * u + 1] = h.y + r.y;
                    }
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        load_scales<NB>(dv[i][u], vst, 16 * i + 4 * t + u);
                        // (0 times a scale that is no number is not 0)
                        if (EDGE && !((col_seen >> (16 * i + 4 * t + u)) & 1))
#pragma unroll
                            for (int b = 0; b < NB / 2; b++) dv[i][u][b] = __float2half2_rn(0.0f);
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) {
                            const __half2 x = __habs2(dv[i][u][b]);
                            top[b] = i + u == 0 ? x : __hmax2(top[b], x);
                        }
                    }
                }
#pragma unroll
                for (int b = 0; b < NB / 2; b++)
#pragma unroll
                    for (int s = 1; s <= 2; s <<= 1) {
                        const uint32_t y = __shfl_xor_sync(FULL, *reinterpret_cast<uint32_t*>(&top[b]), s);
                        top[b] = __hmax2(top[b], *reinterpret_cast<const __half2*>(&y));
                    }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float big = b & 1 ? __high2float(top[b / 2]) : __low2float(top[b / 2]);
                    // 2^e <= big < 2^(e + 1); zero, or no finite scale: e = 0 or 16
                    const int e = big > 0.0f ? min(16, (int)(__float_as_uint(big) >> 23) - 127) : 0;
                    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                    float up[2];  // of columns 2t, 2t + 1 (columns may see different keys)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        up[j] = EDGE ? __uint_as_float((uint32_t)(127 + __shfl_sync(FULL, e, 8 * t + 4 * j)) << 23)
                                     : __uint_as_float((uint32_t)(127 + e) << 23);
                    float acc[2][4] = {};
#pragma unroll
                    for (int i = 0; i < MT; i++) {
                        uint32_t bh[2];
                        [[maybe_unused]] uint32_t bl[2];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const __half2 *d0 = dv[i][2 * u], *d1 = dv[i][2 * u + 1];
                            const float x = w[i][2 * u] * ((b & 1 ? __high2float(d0[b / 2]) : __low2float(d0[b / 2])) * down);
                            const float y = w[i][2 * u + 1] * ((b & 1 ? __high2float(d1[b / 2]) : __low2float(d1[b / 2])) * down);
                            bh[u] = pack2(x, y);
                            if constexpr (LO) bl[u] = rest2(x, y, bh[u]);
                            if constexpr (PACK) {
                                const uint32_t r = rest2(x, y, bh[u]);
                                if (g >= 4) bh[u] = r;
                            }
                        }
                        uint32_t va[2][4];
                        if constexpr (TYPE == KV_Q8_0) {
                            uint32_t x4[4];
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                x4[j] = *reinterpret_cast<const uint32_t*>(
                                            vt + KT::off(16 * i + 4 * t + j, 2 * b + (g >> 2), true) + (g & 3) * 4) ^
                                        0x80808080u;
#pragma unroll
                            for (int u = 0; u < 2; u++) {  // keys 4t + 2u, 4t + 2u + 1; dims 4g … 4g + 3 of the block
                                const uint32_t x = __byte_perm(x4[2 * u], x4[2 * u + 1], 0x5140);
                                const uint32_t y = __byte_perm(x4[2 * u], x4[2 * u + 1], 0x7362);
                                va[0][2 * u] = bytes_h2(x, 0x4140, H2_1152), va[0][2 * u + 1] = bytes_h2(x, 0x4342, H2_1152);
                                va[1][2 * u] = bytes_h2(y, 0x4140, H2_1152), va[1][2 * u + 1] = bytes_h2(y, 0x4342, H2_1152);
                            }
                        } else {
                            uint32_t x4[4];
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                x4[j] = *reinterpret_cast<const uint16_t*>(vt + KT::off(16 * i + 4 * t + j, b, true) + g * 2);
#pragma unroll
                            for (int u = 0; u < 2; u++) {  // dims 2g, 2g + 1 (low nibbles) and 16 + 2g, 17 + 2g (high)
                                const uint32_t x = __byte_perm(x4[2 * u], x4[2 * u + 1], 0x5410);
                                va[0][2 * u] = nibbles_h2<false>(x), va[0][2 * u + 1] = nibbles_h2<false>(x >> 8);
                                va[1][2 * u] = nibbles_h2<true>(x), va[1][2 * u + 1] = nibbles_h2<true>(x >> 8);
                            }
                        }
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            mma16816(acc[s], va[s], bh[0], bh[1]);
                            if constexpr (LO) mma16816(acc[s], va[s], bl[0], bl[1]);
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            o[2 * b + s][j] = fmaf(o[2 * b + s][j], alpha[j & 1], acc[s][j] * up[j & 1]);
                }
            }
        };

        for (; ct < seg_end; ct += TEAMS, done++) {
            cp_wait<STAGES - 2>();
            if constexpr (WR == 1)
                __syncwarp();
            else
                bar_sync(1 + team, WR * 32);
            load();  // into the stage that was computed last
            const uint8_t* st = ring + done % STAGES * KT::STAGE;
            // whether every row sees every key of the tile
            const int v0 = (ct - cc.first) * KEYS, v1 = v0 + KEYS;
            bool edge = v1 > sp.nv;
            if (many && !edge && v1 > sp.ns) {
                const int p0 = sp.position(v0), p1 = sp.position(v1 - 1);
                edge = v0 < sp.ns || p1 >= sp.pos + (a.parent ? 0 : 1) ||
                       (c.window && p0 <= sp.pos + sp.m - 1 - c.window && p1 >= c.sinks);
            }
            if (edge)
                compute(ct, st, std::true_type{});
            else
                compute(ct, st, std::false_type{});
        }

        // ---- the teams' parts joined: the last teams' into the first's, at most four warps' at a time ----
#pragma unroll
        for (int j = 0; j < 2; j++) {
            l[j] += __shfl_xor_sync(FULL, l[j], 4);
            l[j] += __shfl_xor_sync(FULL, l[j], 8);
            l[j] += __shfl_xor_sync(FULL, l[j], 16);
        }
        if constexpr (PACK) {  // the lo halves' columns to the hi halves'
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[d][j] += __shfl_xor_sync(FULL, o[d][j], 2);
        }
        auto fold = [&](float* mo, float* lo, float f0[2], float f1[2]) {  // weights of the own and the other part
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float mn = fmaxf(m[j], mo[j]), safe = mn == -INFINITY ? 0.0f : mn;
                f0[j] = ex2(m[j] - safe), f1[j] = ex2(mo[j] - safe);
                l[j] = l[j] * f0[j] + lo[j] * f1[j];
                m[j] = mn;
            }
        };
        for (int n = TEAMS; n > 1;) {
            const int give = min(n / 2, 4 / WR);  // teams n - give … n - 1 into teams 0 … give - 1
            if (team >= n - give && team < n) {
                const int w = warp - (n - give) * WR;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) joined[(w * (D / 4) + 4 * d + j) * 32 + lane] = o[d][j];
                if (g == 0) {
                    s_ml[w][2 * t] = m[0], s_ml[w][2 * t + 1] = m[1];
                    s_ml[w][8 + 2 * t] = l[0], s_ml[w][8 + 2 * t + 1] = l[1];
                }
            }
            __syncthreads();
            if (team < give) {
                float mo[2] = {s_ml[warp][2 * t], s_ml[warp][2 * t + 1]};
                float lo[2] = {s_ml[warp][8 + 2 * t], s_ml[warp][8 + 2 * t + 1]}, f0[2], f1[2];
                fold(mo, lo, f0, f1);
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[d][j] = o[d][j] * f0[j & 1] + joined[(warp * (D / 4) + 4 * d + j) * 32 + lane] * f1[j & 1];
            }
            __syncthreads();
            n -= give;
        }
        // ---- the output, or this CTA's part of it ----
        auto dim = [&](int d, int up) {  // the dim of tile d's row g (up = 0) or g + 8
            if (TYPE == KV_F16) return 16 * d + 8 * up + g;
            if (TYPE == KV_Q8_0) return 32 * (d >> 1) + 4 * g + 2 * (d & 1) + up;
            return 32 * (d >> 1) + 16 * (d & 1) + 2 * g + up;
        };
        auto put = [&](int w, int d, const float* x, const float* ll) {  // rows 8 w + 2t, 8 w + 2t + 1
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int r = 8 * w + 2 * t + j;
                if (r >= rows) continue;
                T* op = static_cast<T*>(a.out) + cc.b * a.o_slot + (r / G) * a.o_row + (cc.h * G + r % G) * a.o_head;
                const float inv = ll[j] == 0.0f ? 0.0f : 1.0f / ll[j];
                op[dim(d, 0)] = (T)(ll[j] == 0.0f ? 0.0f : x[j] * inv);
                op[dim(d, 1)] = (T)(ll[j] == 0.0f ? 0.0f : x[j + 2] * inv);
            }
        };
        if (seg_end - seg == cc.tiles) {
            if (team == 0)
#pragma unroll
                for (int d = 0; d < DT; d++) put(wr, d, o[d], l);
        } else {
            // parts: [2 CTAs][WR][D / 4 registers][32 lanes], then [WR][m 8, l 8]; the pair's first CTA holds it as its
            // last pair (part 1), the others as their first (part 0)
            constexpr int PART = WR * (D * 8 + 16);
            uint32_t* tickets = static_cast<uint32_t*>(a.work);
            float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + KV_TICKETS);
            const int c0 = cut.owner(cc.first), c1 = cut.owner(cc.first + cc.tiles - 1);
            float* mine = parts + (size_t)(2 * cta + (cta == c0)) * PART;
            if (team == 0) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) __stcg(&mine[(wr * (D / 4) + 4 * d + j) * 32 + lane], o[d][j]);
                if (g == 0) {
                    float* ml = mine + WR * D * 8 + wr * 16;
                    __stcg(&ml[2 * t], m[0]), __stcg(&ml[2 * t + 1], m[1]);
                    __stcg(&ml[8 + 2 * t], l[0]), __stcg(&ml[8 + 2 * t + 1], l[1]);
                }
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool last = atomicAdd(&tickets[c0], 1u) == (uint32_t)(c1 - c0);
                if (last) tickets[c0] = 0;
                __threadfence();
                s_last = last;
            }
            __syncthreads();
            if (s_last) {
                for (int w = warp; w < WR * DT; w += KA_WARPS) {  // (rows 8 r …, tile d) in the CTAs' order
                    const int r = w / DT, d = w % DT;
                    float mx[2] = {-INFINITY, -INFINITY}, ll[2] = {0.0f, 0.0f}, x[4] = {};
                    auto ml_of = [&](int i) { return parts + (size_t)(2 * i + (i == c0)) * PART + WR * D * 8 + r * 16; };
#pragma unroll 8
                    for (int i = c0; i <= c1; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++) mx[j] = fmaxf(mx[j], __ldcg(&ml_of(i)[2 * t + j]));
#pragma unroll
                    for (int j = 0; j < 2; j++) mx[j] = mx[j] == -INFINITY ? 0.0f : mx[j];
#pragma unroll 4  // (the loads of several parts in flight)
                    for (int i = c0; i <= c1; i++) {
                        const float* q = parts + (size_t)(2 * i + (i == c0)) * PART + (r * (D / 4) + 4 * d) * 32 + lane;
                        float f[2];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            f[j] = ex2(__ldcg(&ml_of(i)[2 * t + j]) - mx[j]);
                            ll[j] += __ldcg(&ml_of(i)[8 + 2 * t + j]) * f[j];
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) x[j] += __ldcg(&q[32 * j]) * f[j & 1];
                    }
                    put(r, d, x, ll);
                }
            }
        }
        seg = seg_end;
        if (many && seg < end) __syncthreads();  // (the rows' table is the next pair's)
    }
    cp_wait<0>();
}

template <int TYPE, int D, int WR, bool PACK, class T>
static cudaError_t launch_team(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    constexpr int SMEM = KA_WARPS * KA_RING + 4 * D * 8 * 4;
    static PerDeviceOnce once;
    once([] {
        cudaFuncSetAttribute(k_kv_attn<TYPE, D, WR, PACK, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    });
    return kv_launch(k_kv_attn<TYPE, D, WR, PACK, T>, dim3(a.num_sms), KA_THREADS, SMEM, st, pdl, a);
}
template <int TYPE, int D, class T>
static cudaError_t launch_rows(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    const int rows = a.r.T * (a.n_head / a.c.n_kv);
    if constexpr (sizeof(T) == 4)
        if (rows <= 4) return launch_team<TYPE, D, 1, true, T>(st, a, pdl);
    if (rows <= 8) return launch_team<TYPE, D, 1, false, T>(st, a, pdl);
    if (rows <= 16) return launch_team<TYPE, D, 2, false, T>(st, a, pdl);
    return launch_team<TYPE, D, 4, false, T>(st, a, pdl);
}
template <int TYPE>
static cudaError_t launch_type(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    if (a.c.d == 128)
        return a.half ? launch_rows<TYPE, 128, __half>(st, a, pdl) : launch_rows<TYPE, 128, float>(st, a, pdl);
    return a.half ? launch_rows<TYPE, 64, __half>(st, a, pdl) : launch_rows<TYPE, 64, float>(st, a, pdl);
}

// tickets, two parts for each CTA (of heads of 128, four warps to a team)
size_t kv_attention_few_work(int num_sms) { return KV_TICKETS + (size_t)num_sms * 2 * 4 * (128 * 8 + 16) * 4; }
static cudaError_t launch_few(cudaStream_t st, const KvAttnArgs& all, bool pdl) {
    for (int b = 0; b < all.c.n_slot; b += KA_LINE) {
        const KvAttnArgs a = kv_slots(all, b, min(KA_LINE, all.c.n_slot - b));
        const bool one = a.c.type != KV_F16 && a.r.T * (a.n_head / a.c.n_kv) <= KV_ONE_ROWS;
        const cudaError_t e = one                   ? launch_kv_attention_one(st, a, pdl)
                              : a.c.type == KV_F16  ? launch_type<KV_F16>(st, a, pdl)
                              : a.c.type == KV_Q8_0 ? launch_type<KV_Q8_0>(st, a, pdl)
                                                    : launch_type<KV_Q4_0>(st, a, pdl);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

static bool is_few(const KvAttnArgs& a) { return (long)a.r.T * (a.n_head / a.c.n_kv) <= KA_ROWS; }
cudaError_t launch_kv_attention(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    return is_few(a) ? launch_few(st, a, pdl) : launch_kv_attention_many(st, a, pdl);
}
size_t kv_attention_work_bytes(int num_sms) { return max(kv_attention_few_work(num_sms), kv_attention_many_work(num_sms)); }

}  // namespace ocr
