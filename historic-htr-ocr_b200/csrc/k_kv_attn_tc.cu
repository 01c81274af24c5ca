// k_kv_attn_tc.cu — attention of many rows per kv head (a prompt's rows, a wide tree of drafts) over a KV cache
// (kv.cuh), on the 5th-generation tensor cores. The formula is k_kv_attn.cu's.
//
// A CTA takes 128 (row, query head) pairs of a kv head (the pairs of a row side by side, so K and V are read once for
// the whole group) against the keys that any of them sees, in tiles of 128 keys. Bound: the tensor cores (f32 rows),
// the exponentials (f16 rows: 16 a clock and SM against 128 x 128 of a tile).
//
// Products: S = Q K^T (M = N = 128, both operands in shared memory), O += P V (A = P in TMEM, written over S in place;
// B = V in shared memory, MN-major), f16 operands, f32 sums in TMEM. Exactness: f32 queries and P are f16 hi + lo (22 bits);
// f16 queries are exact, and P is rounded to f16 as the output is. f16 keys and values are exact; a quantised value
// q d (at most 19 bits) splits exactly into f16 hi + lo, so S = Q_hi K_hi + Q_lo K_hi + Q_hi K_lo, and P V alike, carry
// the f32 product to 2^-22. A row's query is scaled by a power of two (its lo part stays in f16's range), a tile's
// scales by a power of two 2^-e, e from the tile's largest: S takes 2^e back with the row's factor; for V the score
// itself takes e as an addend, so that P carries 2^e and the row's reference bounds both.
//
// Softmax: online. Two warpgroups take the tiles in turn, each with sums, reference and O of its own (joined at the
// end), so one's exponentials run beside the other's products. The reference moves when a tile's maximum passes it by
// 2^6 (then O is rescaled in TMEM); weights stay below 2^14.
//
// Roles (512 threads, so that each has 128 registers): warps 0-3 and 4-7 the two softmax groups, a row per thread, one
// thread of each issuing the group's products (P V of its tile, then Q K^T of its next); warps 8-15 stage K and V: raw
// loads one tile ahead in registers, quants to f16 (operands in the 128-byte swizzle). K runs a
// tile ahead of V: the next K is staged during P V, V during Q K^T, so one stage of each keeps the tensor cores fed.
// Every wait is bounded: a role that gives up sets a flag, the others follow, and no copy is in flight (the staging is
// plain loads and stores).
//
// The work: as in k_kv_attn.cu, the tiles of all (slot, row block, kv head) triples form a line cut evenly over the
// SMs, triples in several CTAs joined by the last to arrive; past KV_LINE (slot, row block) pairs a CTA takes one
// triple, longest first.
#include "kv_attn.cuh"
#include "tc.cuh"

namespace ocr {

constexpr int KC_M = 128, KC_KEYS = 128;
constexpr int KC_LOADERS = 8;
constexpr int KC_THREADS = (8 + KC_LOADERS) * 32;
constexpr int KC_RING = 4;  // tiles whose exponents and marks are kept
constexpr float KC_LAG = 6.0f, KC_BIAS = 8.0f;

template <int BYTES>
struct KcWord;
template <>
struct KcWord<16> {
    using type = uint4;
};
template <>
struct KcWord<8> {
    using type = uint2;
};
template <>
struct KcWord<4> {
    using type = uint32_t;
};
template <int TYPE, int D, class T>
struct KcPlan {
    static constexpr bool LO = sizeof(T) == 4, QN = TYPE != KV_F16;
    static constexpr int NB = D / KV_BLOCK, ROW = kv_row_bytes(TYPE, D);
    static constexpr uint32_t Q_BYTES = KC_M * D * 2, T_BYTES = KC_KEYS * D * 2;  // one f16 operand of Q; of K or V
    static constexpr int PARTS = QN ? 2 : 1;                                      // hi (and lo) of K and V
    static constexpr int NS = QN && D == 128 ? 1 : 2;                             // stages
    static constexpr uint32_t SMEM = (LO ? 2 : 1) * Q_BYTES + 2 * NS * PARTS * T_BYTES + 1024;
    // the joined parts: [D][128] sums, [128] references, [128] weights' sums
    static constexpr int PART = (D + 2) * KC_M;
};

// Barriers: a waiter must meet every completion of its barrier in turn (a parity tells only one from the next), so what
// a softmax group waits for is kept per group (tile n is group n % 2's): kfull, vfull, sfull, odone. The staging meets
// every tile: kempty and vempty are kept per stage.
template <int NB>
struct KcShared {
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], odone[2], xfull[KC_RING], mdone[2];
    uint32_t tmem;
    int abort_flag, last;
    int prefix[KV_LINE + 1], wsum[KC_THREADS / 32];
    float fac[KC_M];             // the rows' factors on S
    float ml[2][2][KC_M];        // the groups' references and sums
    int ex[KC_RING][2];          // the tiles' exponents of K and V
    uint32_t bad[KC_RING][4];    // keys of an edge tile whose values are not all finite
    uint32_t red[KC_RING][KC_LOADERS];
    __align__(8) __half scale[KC_RING][2][KC_KEYS][NB];
    int parent[KV_TREE_MAX], depth[KV_TREE_MAX];
};

__device__ __forceinline__ uint32_t kc_sw(int r, int p) { return (uint32_t)r * 128u + (uint32_t)((p ^ (r & 7)) << 4); }

__device__ __forceinline__ bool kc_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
    for (uint32_t i = 0; i < MBAR_TRIES; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    dev_error(err, DEV_TIMEOUT);
    return false;
}
// the same for a whole warp, with one answer: TMEM accesses are the warp's together, none of its lanes may leave alone
__device__ __forceinline__ bool kc_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
    return __all_sync(FULL, kc_wait(bar, parity, abort_flag, err));
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    tmem_ld16(taddr, r);
    tmem_ld16(taddr + 16, r + 16);
}
__device__ __forceinline__ uint32_t h2mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// a b - c, rounded once: the rest of a product past its rounding c
__device__ __forceinline__ uint32_t h2rest(uint32_t a, uint32_t b, uint32_t c) {
    const uint32_t n = c ^ 0x80008000u;
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&n));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2max(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ bool h2_not_finite(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// ---- the staging of a tile, by 256 threads: raw rows to registers, later to operands ------------------------------------
// K and V alike: rows of 64 dims (128 bytes, swizzled) in D / 64 halves of 128 keys — K is read along the dims (K-major),
// V along the keys (MN-major), from the same layout. A warp's load covers four whole 128-byte lines; the lanes stand so
// that the eight of a store's phase (one or more keys, units side by side) meet all eight 16-byte pieces of a row.
template <int TYPE, int D>
struct KcRaw {
    static constexpr bool QN = TYPE != KV_F16;
    static constexpr int NB = D / KV_BLOCK, ROW = kv_row_bytes(TYPE, D);
    static constexpr int UPK = ROW / 16;                               // 16-byte units of a key
    static constexpr int KU = KC_KEYS * UPK / (KC_LOADERS * 32);       // units of a thread
    static constexpr int UG = TYPE == KV_F16 ? 8 : TYPE == KV_Q8_0 ? 4 : 2;  // units of a key among eight lanes
    static constexpr int PC = 8 / UG;                                  // 16-byte pieces of f16 from a unit
    static constexpr int KPW = 8 / UG * 4 / (D / 64);                  // keys of a warp's load
    static constexpr int STEP = KC_LOADERS * KPW;                      // keys from one unit of a thread to its next
    uint4 k[KU], v[KU];
    uint32_t ex[QN ? NB / 2 : 1];  // the scales of one key: K's for threads 0 … 127, V's for the others

    __device__ static __forceinline__ void place(int lw, int lane, int& key, int& u) {  // of the thread's first unit
        const int q = lane >> 3, l = lane & 7;
        key = lw * KPW + 8 / UG * (q / (D / 64)) + l / UG;
        u = UG * (q % (D / 64)) + l % UG;
    }
    // The tile at key v. Where its 128 rows lie one after another (all but the tiles at an end of the span, of the sinks
    // or of a ring), the addresses are one base and constants.
    struct Tile {
        size_t row;  // of the first key
        int v0;
        bool run;
        __device__ __forceinline__ Tile(const KvView& c, const KvSpan& s, size_t base, int v) : v0(v) {
            const int r = kv_row(c, s.position(v)), last = v + KC_KEYS - 1;
            run = last < s.nv && (v >= s.ns || last < s.ns) && kv_row(c, s.position(last)) - r == KC_KEYS - 1;
            row = base + r;
        }
    };
    __device__ __forceinline__ void load(uint4* x, const uint8_t* data, const KvView& c, const KvSpan& s, size_t base,
                                         const Tile& t, int lw, int lane) {
        int key, u;
        place(lw, lane, key, u);
        if (t.run) {
            const uint8_t* p = data + (t.row + key) * ROW + u * 16;
#pragma unroll
            for (int i = 0; i < KU; i++) x[i] = *reinterpret_cast<const uint4*>(p + i * STEP * ROW);
            return;
        }
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int w = t.v0 + key + i * STEP;
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (w < s.nv) x[i] = *reinterpret_cast<const uint4*>(data + (base + kv_row(c, s.position(w))) * ROW + u * 16);
        }
    }
    __device__ __forceinline__ void load_scales(const KvView& c, const KvSpan& s, size_t base, const Tile& t, int lt) {
        if constexpr (QN) {
            const int w = t.v0 + (lt & (KC_KEYS - 1));
#pragma unroll
            for (int j = 0; j < NB / 2; j++) ex[j] = 0u;
            if (w < s.nv) {
                const size_t row = t.run ? t.row + (lt & (KC_KEYS - 1)) : base + kv_row(c, s.position(w));
                const uint32_t* p = reinterpret_cast<const uint32_t*>((lt < KC_KEYS ? c.ks : c.vs) + row * NB);
#pragma unroll
                for (int j = 0; j < NB / 2; j++) ex[j] = p[j];
            }
        }
    }
    // The operands, values times 2^-e. `bad` (an edge tile's V): what is not finite becomes zero and its key is marked.
    __device__ static __forceinline__ void store(const uint4* x, uint8_t* hi, uint8_t* lo, const __half* scale, int e,
                                                 uint32_t* bad, int lw, int lane) {
        const float down = exp2i(-e);
        int key0, u;
        place(lw, lane, key0, u);
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int key = key0 + i * STEP;
            if constexpr (!QN) {
                uint4 y = x[i];
                if (bad && (h2_not_finite(y.x) || h2_not_finite(y.y) || h2_not_finite(y.z) || h2_not_finite(y.w))) {
                    atomicOr(&bad[key >> 5], 1u << (key & 31));
                    y = make_uint4(0u, 0u, 0u, 0u);
                }
                *reinterpret_cast<uint4*>(hi + (u >> 3) * (KC_KEYS * 128) + kc_sw(key, u & 7)) = y;
            } else {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                float f = __half2float(scale[key * NB + (TYPE == KV_Q8_0 ? u >> 1 : u)]);
                if (bad && !(fabsf(f) <= 65504.0f)) {
                    atomicOr(&bad[key >> 5], 1u << (key & 31));
                    f = 0.0f;
                }
                const uint32_t d = pack2(f * down, f * down);
                uint32_t q[4 * PC];  // pairs of dims in order
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (TYPE == KV_Q8_0) {
                        q[2 * j] = bytes_h2(w[j] ^ 0x80808080u, 0x4140, H2_1152);
                        q[2 * j + 1] = bytes_h2(w[j] ^ 0x80808080u, 0x4342, H2_1152);
                    } else {
                        const uint32_t a = __byte_perm(w[j], 0u, 0x4140), b = __byte_perm(w[j], 0u, 0x4342);
                        q[2 * j] = nibbles_h2<false>(a), q[2 * j + 1] = nibbles_h2<false>(b);
                        q[8 + 2 * j] = nibbles_h2<true>(a), q[8 + 2 * j + 1] = nibbles_h2<true>(b);
                    }
                }
#pragma unroll
                for (int j = 0; j < PC; j++) {
                    const int pc = PC * u + j;
                    const uint32_t at = (pc >> 3) * (KC_KEYS * 128) + kc_sw(key, pc & 7);
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        h[y] = h2mul(q[4 * j + y], d);
                        l[y] = h2rest(q[4 * j + y], d, h[y]);
                    }
                    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
        }
    }
};

template <int TYPE, int D, class T>
__global__ void __launch_bounds__(KC_THREADS, 1) k_kv_attn_tc(const __grid_constant__ KvAttnArgs a, int blocks, int line) {
    using P = KcPlan<TYPE, D, T>;
    using Raw = KcRaw<TYPE, D>;
    constexpr int NS = P::NS;
    extern __shared__ uint8_t sm_raw[];
    __shared__ __align__(8) KcShared<P::QN ? P::NB : 1> sh;
    volatile int* abort_flag = &sh.abort_flag;
    const KvView& c = a.c;
    int* err = a.err;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.n_head / c.n_kv;
    uint8_t* Qh = sm_raw + ((1024u - (smem_u32(sm_raw) & 1023u)) & 1023u);
    uint8_t* Ql = Qh + P::Q_BYTES;
    uint8_t* Kr = Qh + (P::LO ? 2 : 1) * P::Q_BYTES;
    uint8_t* Vr = Kr + NS * P::PARTS * P::T_BYTES;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.kfull[i], KC_LOADERS);
            mbar_init(&sh.kempty[i], 1);
            mbar_init(&sh.vfull[i], KC_LOADERS);
            mbar_init(&sh.vempty[i], 1);
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.mdone[i], 1);
            mbar_init(&sh.odone[i], 1);
        }
        for (int i = 0; i < KC_RING; i++) mbar_init(&sh.xfull[i], 1);
        sh.abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 0) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    pdl_wait();

    // ---- the line: exclusive sums of the tiles of every (slot, row block) ----
    const int entries = c.n_slot * blocks;
    auto rows_of_block = [&](int blk, int& t0, int& t1) { t0 = blk * KC_M / G, t1 = (blk * KC_M + KC_M - 1) / G + 1; };
    bool idle_rows = false;
    for (int b = tid; b < c.n_slot; b += KC_THREADS) idle_rows |= a.r.rows(c, b, err) < a.r.T;
    int total = 0;
    if (line) {
        int x = 0;
        if (tid < entries) {  // (at most KV_LINE of them)
            int t0, t1;
            rows_of_block(tid % blocks, t0, t1);
            KvSpan s;
            s.set(a, tid / blocks, t0, t1);
            x = (s.nv + KC_KEYS - 1) / KC_KEYS * c.n_kv;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sh.wsum[warp] = x;
        __syncthreads();
        for (int w = 0; w < warp; w++) x += sh.wsum[w];
        if (tid < entries) sh.prefix[tid + 1] = x;
        if (tid == 0) sh.prefix[0] = 0;
        for (int w = 0; w < KC_THREADS / 32; w++) total += sh.wsum[w];
    }
    tc_fence_before();
    const bool some_idle = __syncthreads_or(idle_rows);
    tc_fence_after();
    if (some_idle) {  // rows that are not in use are zeros
        const long n = (long)c.n_slot * a.r.T * a.n_head;
        for (long i = (long)blockIdx.x * (KC_THREADS / 32) + warp; i < n; i += (long)gridDim.x * (KC_THREADS / 32)) {
            const int h = (int)(i % a.n_head), r = (int)(i / a.n_head % a.r.T), b = (int)(i / a.n_head / a.r.T);
            if (r < a.r.rows(c, b, nullptr)) continue;
            T* o = static_cast<T*>(a.out) + b * a.o_slot + r * a.o_row + h * a.o_head;
            for (int d = lane; d < D; d += 32) o[d] = (T)0.0f;
        }
    }
    const uint32_t tmem = sh.tmem;
    const int n_cta = line ? min((int)gridDim.x, total) : (int)gridDim.x;
    const int cta = blockIdx.x;
    KvLine cut;
    cut.cut(total, n_cta);
    int begin = 0, end = 0;
    KvCursor cc;
    if (line) {
        if (cta < n_cta) begin = cut.part(cta), end = cut.part(cta + 1);
    } else {  // one triple, the last row blocks (the longest) first
        const int per = c.n_slot * c.n_kv;
        const int blk = blocks - 1 - cta / per, b = cta % per / c.n_kv;
        int t0, t1;
        rows_of_block(blk, t0, t1);
        KvSpan s;
        s.set(a, b, t0, t1);
        cc.b = b * blocks + blk;
        cc.h = cta % c.n_kv;
        cc.first = 0;
        cc.tiles = (s.nv + KC_KEYS - 1) / KC_KEYS;
        end = cc.tiles;
    }

    int n0 = 0;          // tiles of this CTA before the triple
    bool any_mma = false;  // (the issuing threads)
    for (int seg = begin; seg < end;) {
        if (line) cc.at(seg, sh.prefix, entries, c.n_kv);
        const int slot = cc.b / blocks, blk = cc.b % blocks;
        int t0, t1;
        rows_of_block(blk, t0, t1);
        KvSpan sp;
        sp.set(a, slot, t0, t1);
        const int seg_end = min(end, cc.first + cc.tiles), N = seg_end - seg;
        const int r0 = blk * KC_M, rows = min(KC_M, sp.m * G - r0);
        const size_t base = kv_index(c, slot, cc.h, 0);
        // whether some row of the block does not see some key of the tile
        auto edge_of = [&](int v0) {
            if (v0 + KC_KEYS > sp.nv) return true;
            if (v0 + KC_KEYS <= sp.ns) return false;
            const int p0 = sp.position(v0), p1 = sp.position(v0 + KC_KEYS - 1);
            const int lowest = sp.pos + (a.parent ? -1 : t0), highest = sp.pos + (a.parent ? sp.m : min(t1, sp.m)) - 1;
            return v0 < sp.ns || p1 > lowest || (c.window && p0 <= highest - c.window && p1 >= c.sinks);
        };
        if (a.parent && tid < sp.m) sh.parent[tid] = a.parent[(size_t)slot * a.r.T + tid];
        // ---- the queries: hi and lo, a row per warp at a time ----
        {
            constexpr int R = KC_M / 16, V = D / 32;  // a lane's dims
            alignas(16) T q[R][V];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int r = warp + 16 * i, row = r0 + r;
                const T* qp = static_cast<const T*>(a.q) + slot * a.q_slot + (row / G) * a.q_row +
                              (cc.h * G + row % G) * a.q_head + lane * V;
                using Word = typename KcWord<V * sizeof(T)>::type;
                Word w = {};
                if (r < rows) w = *reinterpret_cast<const Word*>(qp);
                *reinterpret_cast<Word*>(q[i]) = w;
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int r = warp + 16 * i;
                float x[V];
                float f = a.scale * LOG2E;
#pragma unroll
                for (int j = 0; j < V; j++) x[j] = (float)q[i][j];
                if constexpr (P::LO) {  // the row's largest to 2^10 … 2^11
                    float big = 0.0f;
#pragma unroll
                    for (int j = 0; j < V; j++) big = fmaxf(big, fabsf(x[j]));
                    big = warp_max(big);
                    const int e = big > 0.0f && big <= 3.4028234e38f ? min(100, 137 - (int)(__float_as_uint(big) >> 23)) : 0;
                    f *= exp2i(-e);
#pragma unroll
                    for (int j = 0; j < V; j++) x[j] *= exp2i(e);
                }
                if (lane == 0) sh.fac[r] = f;
                const int byte = lane * (D / 16);  // of the row's D f16
                const uint32_t at = (byte >> 7) * (KC_M * 128) + kc_sw(r, (byte >> 4) & 7) + (byte & 15);
#pragma unroll
                for (int j = 0; j < V / 2; j++) {
                    const uint32_t h = pack2(x[2 * j], x[2 * j + 1]);
                    *reinterpret_cast<uint32_t*>(Qh + at + 4 * j) = h;
                    if constexpr (P::LO) *reinterpret_cast<uint32_t*>(Ql + at + 4 * j) = rest2(x[2 * j], x[2 * j + 1], h);
                }
            }
            fence_proxy_async();
        }
        __syncthreads();
        if (a.parent) {
            if (tid < sp.m) {
                sh.depth[tid] = kv_depth(tid, sh.parent, err);
            }
            __syncthreads();
        }

        if (warp >= 8 && warp < 16) {
            // ---- the staging: K of tile i + 1, then V of tile i ----
            const int lw = warp - 8, lt = tid - 256;
            Raw raw{};
            const int vb = (seg - cc.first) * KC_KEYS;
            bool ok = true;  // (a thread that gave up still meets the others at every tile's barrier)
            auto put_k = [&](int i) {  // → the exponent of V's tile
                const int n = n0 + i, st = n % NS, x = n % KC_RING;
                int eK = 0, eV = 0;
                if (lt < 4) sh.bad[x][lt] = 0u;
                if constexpr (P::QN) {
                    uint32_t big = 0u;
#pragma unroll
                    for (int j = 0; j < P::NB / 2; j++) {
                        big = h2max(big, raw.ex[j] & 0x7fff7fffu);
                        reinterpret_cast<uint32_t*>(sh.scale[x][lt >> 7][lt & 127])[j] = raw.ex[j];
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) big = h2max(big, __shfl_xor_sync(FULL, big, o));
                    if (lane == 0) sh.red[x][lw] = big;
                }
                bar_sync(2, KC_LOADERS * 32);
                if constexpr (P::QN) {
                    auto exponent = [&](int w) {
                        uint32_t b = sh.red[x][w];
#pragma unroll
                        for (int j = 1; j < KC_LOADERS / 2; j++) b = h2max(b, sh.red[x][w + j]);
                        const __half2 h = *reinterpret_cast<const __half2*>(&b);
                        const float f = fmaxf(__low2float(h), __high2float(h));
                        return f > 0.0f ? min(16, (int)(__float_as_uint(f) >> 23) - 127) : 0;
                    };
                    eK = exponent(0);
                    eV = exponent(KC_LOADERS / 2);
                    if (lt == 0) {
                        sh.ex[x][0] = eK, sh.ex[x][1] = eV;
                        mbar_arrive(&sh.xfull[x]);
                    }
                }
                ok = ok && (n < NS || kc_wait(&sh.kempty[st], (n / NS - 1) & 1, abort_flag, err));
                uint8_t* kh = Kr + st * P::PARTS * P::T_BYTES;
                if (ok) Raw::store(raw.k, kh, kh + P::T_BYTES, sh.scale[x][0][0], eK, nullptr, lw, lane);
                fence_proxy_async();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&sh.kfull[n & 1]);
                if (i + 1 < N) {
                    const typename Raw::Tile t(c, sp, base, vb + (i + 1) * KC_KEYS);
                    raw.load(raw.k, c.k, c, sp, base, t, lw, lane);
                    raw.load_scales(c, sp, base, t, lt);
                }
                return eV;
            };
            {
                const typename Raw::Tile first(c, sp, base, vb);
                raw.load_scales(c, sp, base, first, lt);
                raw.load(raw.k, c.k, c, sp, base, first, lw, lane);
                raw.load(raw.v, c.v, c, sp, base, first, lw, lane);
            }
            int eV = put_k(0);
            for (int i = 0; i < N; i++) {
                const int n = n0 + i, st = n % NS, x = n % KC_RING, v0 = vb + i * KC_KEYS;
                const int e = eV;
                if (i + 1 < N) eV = put_k(i + 1);
                ok = ok && (n < NS || kc_wait(&sh.vempty[st], (n / NS - 1) & 1, abort_flag, err));
                uint8_t* vh = Vr + st * P::PARTS * P::T_BYTES;
                if (ok)
                    Raw::store(raw.v, vh, vh + P::T_BYTES, sh.scale[x][1][0], e, edge_of(v0) ? sh.bad[x] : nullptr, lw, lane);
                fence_proxy_async();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&sh.vfull[n & 1]);
                if (i + 1 < N) raw.load(raw.v, c.v, c, sp, base, typename Raw::Tile(c, sp, base, v0 + KC_KEYS), lw, lane);
            }
        } else {
            // ---- the rows: thread r of group wg owns pair r0 + r (TMEM lane r) ----
            const int wg = warp >> 2, r = tid & 127;
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t tS = tmem + lanes + wg * KC_KEYS, tO = tmem + lanes + 256 + wg * 128;
            const int row = min((r0 + r) / G, sp.m - 1);
            KvSight sight;
            if (a.parent)
                kv_draft(c, sp, row, sh.parent, sh.depth, sight);
            else
                sight.rows(c, sp, sp.pos + row, sp.pos + row);
            const float fac0 = sh.fac[r];
            float m = -INFINITY, l = 0.0f;
            // the group's products, by one thread
            const bool issues = (tid & 127) == 0;
            constexpr uint32_t idS = bg_idesc(KC_KEYS), idO = bg_idesc_mn(D);
            auto qk = [&](int n) {
                const int st = n % NS;
                if (!kc_wait(&sh.kfull[wg], (n >> 1) & 1, abort_flag, err)) return;
                tc_fence_after();
                const uint32_t qh = smem_u32(Qh), ql = smem_u32(Ql);
                const uint32_t kh = smem_u32(Kr + st * P::PARTS * P::T_BYTES), kl = kh + P::T_BYTES;
                // the small products first: a sum loses what falls below its last bit at every product added
                constexpr int SMALL = (P::LO ? 1 : 0) + (P::QN ? 1 : 0);
#pragma unroll
                for (int x = 0; x <= SMALL; x++)
#pragma unroll
                    for (int k = 0; k < D / 16; k++) {
                        const uint32_t o = (k >> 2) * (128 * 128) + (k & 3) * 32;
                        const bool lq = P::LO && x == 0, lk = P::QN && x == (P::LO ? 1 : 0);
                        mma_f16(tmem + wg * KC_KEYS, bg_desc((lq ? ql : qh) + o), bg_desc((lk ? kl : kh) + o), idS,
                                x + k > 0 ? 1u : 0u);
                    }
                mma_commit(&sh.sfull[wg]);
                mma_commit(&sh.kempty[st]);
                any_mma = true;
            };
            auto pv = [&](int n, bool fresh) {
                const int st = n % NS;
                if (!kc_wait(&sh.vfull[wg], (n >> 1) & 1, abort_flag, err)) return;
                tc_fence_after();
                const uint32_t vh = smem_u32(Vr + st * P::PARTS * P::T_BYTES), vl = vh + P::T_BYTES;
                const uint32_t tP = tmem + wg * KC_KEYS, tD = tmem + 256 + wg * 128;
#pragma unroll
                for (int k = 0; k < KC_KEYS / 16; k++) {  // 32 keys' P: hi in 16 columns, lo in the next 16
                    const uint32_t p = tP + (k >> 1) * 32 + (k & 1) * 8;
                    const uint64_t bh = bg_desc_mn(vh + k * 2048, KC_KEYS * 128), bl = bg_desc_mn(vl + k * 2048, KC_KEYS * 128);
                    mma_f16_ts(tD, p, bh, idO, (!fresh || k > 0) ? 1u : 0u);
                    if constexpr (P::LO) mma_f16_ts(tD, p + 16, bh, idO, 1u);
                    if constexpr (P::QN) mma_f16_ts(tD, p, bl, idO, 1u);
                }
                mma_commit(&sh.odone[wg]);
                mma_commit(&sh.vempty[st]);
            };
            if (issues && ((n0 & 1) ^ wg) < N) qk(n0 + ((n0 & 1) ^ wg));
            __syncwarp();
            auto tile = [&](int i) -> bool {  // the weights of tile i; false: a wait gave up
                const int n = n0 + i, x = n % KC_RING, v0 = (seg - cc.first + i) * KC_KEYS;
                const bool edge = edge_of(v0);
                float fac = fac0, ev = 0.0f;
                if constexpr (P::QN) {
                    if (!kc_wait_warp(&sh.xfull[x], (n / KC_RING) & 1, abort_flag, err)) return false;
                    fac *= exp2i(sh.ex[x][0]);
                    ev = (float)sh.ex[x][1];
                }
                if (!kc_wait_warp(&sh.sfull[wg], (n >> 1) & 1, abort_flag, err)) return false;
                if (edge && !kc_wait_warp(&sh.vfull[wg], (n >> 1) & 1, abort_flag, err)) return false;  // (the marks)
                tc_fence_after();
                // a chunk of 32 scores, what the row does not see taken out
                auto chunk = [&](int ch, uint32_t* s) {
                    tmem_ld32(tS + 32 * ch, s);
                    tmem_wait_ld();
                    if (!edge) return;
                    const uint32_t see = sight.mask(v0 + 32 * ch), bad = sh.bad[x][ch] & see;
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (!((see >> j) & 1)) s[j] = 0xff800000u;
                    if (bad) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if ((bad >> j) & 1) s[j] = 0x7fffffffu;
                    }
                };
                float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                for (int ch = 0; ch < 4; ch++) {
                    uint32_t s[32];
                    chunk(ch, s);
#pragma unroll
                    for (int j = 0; j < 32; j++) mq[j & 3] = fmaxf(mq[j & 3], __uint_as_float(s[j]));
                }
                const float mt = fmaf(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])), fac, ev);
                if (i < 2) {
                    m = mt;
                } else if (__any_sync(FULL, mt > m + KC_LAG)) {
                    // (warp-uniform: TMEM loads and stores are the whole warp's; a row that stays scales by 1)
                    if (!kc_wait_warp(&sh.odone[wg], ((n >> 1) - 1) & 1, abort_flag, err)) return false;
                    tc_fence_after();
                    const bool up = mt > m + KC_LAG;
                    const float f = up ? ex2(m - mt) : 1.0f;
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t o[16];
                        tmem_ld16(tO + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                        tmem_st16(tO + d, o);
                    }
                    l *= f;
                    if (up) m = mt;
                }
                const float ref = ev + KC_BIAS - (m == -INFINITY ? 0.0f : m);
                float sum[2] = {0.0f, 0.0f};
#pragma unroll 1
                for (int ch = 0; ch < 4; ch++) {
                    uint32_t s[32], h[16];
                    chunk(ch, s);
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const float p = ex2(fmaf(__uint_as_float(s[j]), fac, ref));
                        s[j] = __float_as_uint(p);
                        sum[j & 1] += p;
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float p0 = __uint_as_float(s[2 * j]), p1 = __uint_as_float(s[2 * j + 1]);
                        h[j] = pack2(p0, p1);
                        if constexpr (P::LO) s[j] = rest2(p0, p1, h[j]);
                    }
                    tmem_st16(tS + 32 * ch, h);
                    if constexpr (P::LO) tmem_st16(tS + 32 * ch + 16, s);
                }
                l = fmaf(sum[0] + sum[1], exp2i(P::QN ? -(int)ev : 0), l);
                tmem_wait_st();
                return true;
            };
            bool ok = true;  // (a warp that gave up still meets its group at every tile)
            for (int i = (n0 & 1) ^ wg; i < N; i += 2) {
                const int n = n0 + i;
                ok = ok && tile(i);
                tc_fence_before();
                bar_sync(4 + wg, 128);
                if (issues && ok) {
                    tc_fence_after();
                    pv(n, i < 2);
                    // (P lies over S: its product is done before the next S)
                    if (i + 2 < N && kc_wait(&sh.odone[wg], (n >> 1) & 1, abort_flag, err)) qk(n + 2);
                }
                __syncwarp();
            }
            sh.ml[wg][0][r] = m;
            sh.ml[wg][1][r] = l;
            // both groups' products are done: this group's last tile, and the other's
            ok = __all_sync(FULL, ok && *abort_flag == 0);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int last = n0 + N - 1 - ((n0 + N - 1 - w) & 1);  // the last tile of group w
                if (last >= n0 && ok) ok = kc_wait_warp(&sh.odone[w], (last >> 1) & 1, abort_flag, err);
            }
            tc_fence_after();
            bar_sync(3, 256);
            // the row's sums: each group writes half of the dims
            const int w0 = n0 & 1;
            const bool two = N > 1;
            const float ma = sh.ml[w0][0][r], mb = two ? sh.ml[w0 ^ 1][0][r] : -INFINITY;
            const float mx = fmaxf(ma, mb), safe = mx == -INFINITY ? 0.0f : mx;
            const float fa = ex2(ma - safe), fb = ex2(mb - safe);
            const float lt = sh.ml[w0][1][r] * fa + (two ? sh.ml[w0 ^ 1][1][r] * fb : 0.0f);
            const bool whole = N == cc.tiles;
            const int c0 = whole ? 0 : cut.owner(cc.first);
            float* mine = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + KV_TICKETS) +
                          (size_t)(2 * cta + (cta == c0)) * P::PART;
            const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
            // (Q's memory is free: every product is done) the rows of the output, 16-byte pieces moved among eight
            constexpr int ROW = D * sizeof(T);
            if (ok) {
#pragma unroll 1
                for (int d = wg * (D / 2); d < (wg + 1) * (D / 2); d += 16) {
                    uint32_t o[16], o2[16];
                    tmem_ld16(tmem + lanes + 256 + w0 * 128 + d, o);
                    if (two) tmem_ld16(tmem + lanes + 256 + (w0 ^ 1) * 128 + d, o2);
                    tmem_wait_ld();
                    float y[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        y[j] = __uint_as_float(o[j]) * fa;
                        if (two) y[j] = fmaf(__uint_as_float(o2[j]), fb, y[j]);
                    }
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 16; j++) __stcg(&mine[(d + j) * KC_M + r], y[j]);
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) y[j] = lt == 0.0f ? 0.0f : y[j] * inv;
                    constexpr int E = 16 / sizeof(T);  // elements of a piece
#pragma unroll
                    for (int j = 0; j < 16 / E; j++) {
                        uint4 w;
                        if constexpr (P::LO)
                            w = make_uint4(__float_as_uint(y[4 * j]), __float_as_uint(y[4 * j + 1]),
                                           __float_as_uint(y[4 * j + 2]), __float_as_uint(y[4 * j + 3]));
                        else
                            w = make_uint4(pack2(y[8 * j], y[8 * j + 1]), pack2(y[8 * j + 2], y[8 * j + 3]),
                                           pack2(y[8 * j + 4], y[8 * j + 5]), pack2(y[8 * j + 6], y[8 * j + 7]));
                        *reinterpret_cast<uint4*>(Qh + r * ROW + (((d / E + j) ^ (r & 7)) << 4)) = w;
                    }
                }
                if (whole) {
                    bar_sync(3, 256);
                    constexpr int PC = ROW / 16;
                    for (int e = tid; e < rows * PC; e += 256) {
                        const int rr = e / PC, pc = e % PC;
                        T* op = static_cast<T*>(a.out) + slot * a.o_slot + ((r0 + rr) / G) * a.o_row +
                                (cc.h * G + (r0 + rr) % G) * a.o_head;
                        reinterpret_cast<uint4*>(op)[pc] = *reinterpret_cast<const uint4*>(Qh + rr * ROW + ((pc ^ (rr & 7)) << 4));
                    }
                }
                if (!whole && wg == 0) {
                    __stcg(&mine[D * KC_M + r], mx);
                    __stcg(&mine[(D + 1) * KC_M + r], lt);
                }
                if (!whole) __threadfence();
            }
            tc_fence_before();
        }
        __syncthreads();
        tc_fence_after();
        if (*abort_flag) break;
        // ---- a triple that lies in several CTAs: the last of them joins the parts in the CTAs' order ----
        if (N != cc.tiles) {
            const int c0 = cut.owner(cc.first), c1 = cut.owner(cc.first + cc.tiles - 1);
            uint32_t* tickets = static_cast<uint32_t*>(a.work);
            if (tid == 0) {
                const bool last = atomicAdd(&tickets[c0], 1u) == (uint32_t)(c1 - c0);
                if (last) tickets[c0] = 0;
                __threadfence();
                sh.last = last;
            }
            __syncthreads();
            if (sh.last) {
                const int r = tid & 127, d0 = (tid >> 7) * (D / 4);
                const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.work) + KV_TICKETS);
                auto of = [&](int i) { return parts + (size_t)(2 * i + (i == c0)) * P::PART; };
                float mx = -INFINITY, l = 0.0f, y[D / 4] = {};
                for (int i = c0; i <= c1; i++) mx = fmaxf(mx, __ldcg(&of(i)[D * KC_M + r]));
                if (mx == -INFINITY) mx = 0.0f;
                for (int i = c0; i <= c1; i++) {
                    const float* q = of(i);
                    const float f = ex2(__ldcg(&q[D * KC_M + r]) - mx);
                    l = fmaf(__ldcg(&q[(D + 1) * KC_M + r]), f, l);
#pragma unroll
                    for (int d = 0; d < D / 4; d++) y[d] = fmaf(__ldcg(&q[(d0 + d) * KC_M + r]), f, y[d]);
                }
                if (r < rows) {
                    T* op = static_cast<T*>(a.out) + slot * a.o_slot + ((r0 + r) / G) * a.o_row +
                            (cc.h * G + (r0 + r) % G) * a.o_head + d0;
                    const float inv = 1.0f / l;
#pragma unroll
                    for (int d = 0; d < D / 4; d++) op[d] = (T)(l == 0.0f ? 0.0f : y[d] * inv);
                }
            }
        }
        n0 += N;
        seg = seg_end;
    }
    // ---- every product complete before the TMEM is given back ----
    if (warp < 8 && (tid & 127) == 0 && any_mma) {
        mma_commit(&sh.mdone[warp >> 2]);
        mbar_wait(&sh.mdone[warp >> 2], 0, err);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int TYPE, int D, class T>
static cudaError_t launch_tc(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    using P = KcPlan<TYPE, D, T>;
    static PerDeviceOnce once;
    once([] { cudaFuncSetAttribute(k_kv_attn_tc<TYPE, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::SMEM); });
    const int blocks = (int)(((long)a.r.T * (a.n_head / a.c.n_kv) + KC_M - 1) / KC_M);
    const bool line = (long)a.c.n_slot * blocks <= KV_LINE;
    const long grid = line ? a.num_sms : (long)a.c.n_slot * blocks * a.c.n_kv;
    return kv_launch(k_kv_attn_tc<TYPE, D, T>, dim3((unsigned)grid), KC_THREADS, P::SMEM, st, pdl, a, blocks, line ? 1 : 0);
}
template <int TYPE>
static cudaError_t launch_type(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    if (a.c.d == 128) return a.half ? launch_tc<TYPE, 128, __half>(st, a, pdl) : launch_tc<TYPE, 128, float>(st, a, pdl);
    return a.half ? launch_tc<TYPE, 64, __half>(st, a, pdl) : launch_tc<TYPE, 64, float>(st, a, pdl);
}
// tickets, and two parts for each CTA
size_t kv_attention_many_work(const KvAttnArgs& a) { return KV_TICKETS + (size_t)a.num_sms * 2 * (a.c.d + 2) * KC_M * 4; }
cudaError_t launch_kv_attention_many(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    switch (a.c.type) {
        case KV_F16: return launch_type<KV_F16>(st, a, pdl);
        case KV_Q8_0: return launch_type<KV_Q8_0>(st, a, pdl);
        default: return launch_type<KV_Q4_0>(st, a, pdl);
    }
}

}  // namespace ocr
