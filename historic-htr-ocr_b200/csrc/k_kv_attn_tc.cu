// k_kv_attn_tc.cu — attention of many rows per kv head (a prompt's rows, a wide tree of drafts) over a KV cache
// (kv.cuh), on the 5th-generation tensor cores. The formula is k_kv_attn.cu's.
//
// A CTA takes 128 (row, query head) pairs of a kv head (the pairs of a row side by side, so K and V are read once for
// the whole group) against the keys that any of them sees, in tiles of 128 keys. Floor: the tensor cores. What bounds it now
// is the chain S → P → O of one triple (one fits an SM) with the softmax's instructions and the issuing thread's waits in it:
// the tensor pipe is 19 to 33 % busy, issue 36 to 49 % (the three calls below). Measured: 512 f16 rows by 16896 f16 keys, 16
// heads of 64, four slots: 273 us, 386 TFLOP/s; 2214 f32 rows in a window of 512, q8_0, 16 heads of 128: 66 us; 8 trees of 61
// drafts in windows of 8192, q4_0, f16 rows, 32 heads: 218 us.
//
// Products: S = Q K^T (M = N = 128, both operands in shared memory), O += P V (A = P in TMEM, written over S in place;
// B = V in shared memory, MN-major), f16 operands, f32 sums in TMEM. Exactness: f32 queries and P are f16 hi + lo (22 bits);
// f16 queries are exact, and P is rounded to f16 as the output is. f16 keys and values are exact; a quantised value
// q d (at most 19 bits) splits into f16 hi + lo, so S = Q_hi K_hi + Q_lo K_hi + Q_hi K_lo, and P V alike, carry the f32
// product to 2^-22. A row's query is scaled by a power of two (its lo part stays in f16's range); so are the scales d, as
// far up as the products q d fit f16: the split is exact for scales down to 2^-21 (q8_0) or 2^-25 (q4_0) of the largest that
// shares their exponent, and what is smaller is off by 2^-32 of the largest value. K has one exponent, which S takes back
// with the row's factor; V has one for each block of 32 dims and O stands in their units, so an output's accuracy is that
// of its own block (with one exponent for a tile, blocks 2^20 below another had errors of percents).
//
// Softmax: online. Two warpgroups take 64 keys of every tile each, with sums, reference and O of their own (joined at the
// end). S has two places: the next tile's Q K^T runs while the groups turn this tile's S into P, so a group goes from
// one tile's exponentials to the next's without waiting for a product. The reference moves when a tile's maximum passes
// it by 2^6 (then O is rescaled in TMEM); weights stay below 2^14.
//
// Roles (512 threads, 128 registers each): warps 0-3 and 4-7 the two softmax groups, a row per thread; warps 8-14 stage K
// and V: raw loads one tile ahead in registers, quants to f16 (operands in the 128-byte swizzle); one thread of warp 15
// issues the products. K runs a tile ahead of V: the next K is staged during P V, V during Q K^T, so one stage of each
// keeps the tensor cores fed. The staging runs on into the next triple while the softmax groups finish one. Every wait
// is bounded: a role that gives up sets a flag and goes on without work, meeting every barrier, and no copy is in flight
// (the staging is plain loads and stores).
//
// The sums in TMEM lose what falls below their last bit at every product added, towards zero: a million values of one size,
// 31250 products, 2.9 10^-3 of their sum. For f32 rows a group adds its O to a sum of its own in memory after KcPlan::FLUSH
// tiles and starts O afresh — between a tile's weights and the word that they are there, when the products of the tile
// before are nearly done. 666 rows by 2214 f16 keys twice: errors of 1.6 10^-6 of the output instead of 2.3, for 6 us of 62.
// For f16 rows a variant for long caches does so.
//
// The work: as in k_kv_attn.cu, the tiles of all (slot, row block, kv head) triples form a line cut evenly over the
// SMs, triples in several CTAs joined by the last to arrive.
#include "kv_attn.cuh"
#include "tc.cuh"

namespace ocr {

constexpr int KC_M = 128, KC_KEYS = 128;
constexpr int KC_LOADERS = 7;
constexpr int KC_THREADS = (8 + KC_LOADERS + 1) * 32;
constexpr int KC_RING = 4;  // tiles whose exponents and scales are kept
constexpr int KC_MARKS = 8;  // tiles whose marks are kept: looked at two tiles later
constexpr int KC_PIECE = 10;
constexpr float KC_LAG = 6.0f, KC_BIAS = 8.0f;
constexpr int KC_EXP = 15;  // what an exponent has added to it in a byte (f16's own bias; its subnormals count as 2^-15)

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
template <int TYPE, int D, class T, bool LONG>
struct KcPlan {
    static constexpr bool LO = sizeof(T) == 4, QN = TYPE != KV_F16;
    static constexpr bool MOVES = LO || LONG;  // O is moved out of TMEM now and then
    static constexpr int NB = D / KV_BLOCK, ROW = kv_row_bytes(TYPE, D);
    static constexpr uint32_t Q_BYTES = KC_M * D * 2, T_BYTES = KC_KEYS * D * 2;  // one f16 operand of Q; of K or V
    static constexpr int PARTS = QN ? 2 : 1;                                      // hi (and lo) of K and V
    static constexpr int NS = QN && D == 128 ? 1 : 2;                             // stages
    static constexpr uint32_t SMEM = (LO ? 2 : 1) * Q_BYTES + 2 * NS * PARTS * T_BYTES + 1024;
    // a block's quants times its scale d (below 2^(e + 1)) times 2^(HEAD - e) just fit f16
    static constexpr int HEAD = TYPE == KV_Q8_0 ? 8 : 12;
    // tiles between two moves of O: at most 64 products are added to each of its sums in between, for f16 rows 256
    static constexpr int FLUSH = LO ? QN ? 5 : 8 : QN ? 32 : 64;
    // the joined parts: [D][128] sums, [128] references, [128] weights' sums
    static constexpr int PART = (D + 2) * KC_M;
};

// Barriers: a parity tells one completion only from the next, so a waiter must know that the one before has come and that
// the one after has not. Per stage: kfull, kempty, vempty (their waiters meet every tile in turn). Per place of S, tile
// n's being n % 2: sfull, pfull (both groups' warps; a group may be a tile ahead of the products, not two: it needs S, which
// needs both groups' P of two tiles before), odone, vfull.
template <int NB>
struct KcShared {
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pfull[2], odone[2],
        xfull[KC_RING], qfull, mdone;
    uint32_t tmem;
    int abort_flag, last, longest;
    int prefix[KV_LINE + 1], wsum[KC_THREADS / 32];
    float fac[KC_M];             // the rows' factors on S
    float ml[2][3][KC_M];        // the groups' references, sums, and factors on their sums in memory
    float exk[KC_RING];          // the tiles' factors on S: 2^(e - HEAD) of K's scales
    uint32_t exv[KC_RING];       // the exponents of V's blocks as of these tiles, a byte each
    uint32_t bad[KC_MARKS][4];   // keys of an edge tile whose values are not all finite
    uint32_t top[2][NB + 1];     // the largest exponents of a tile's scales, V's blocks' and K's: two in turn
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
__device__ __forceinline__ bool elect_one() {
    uint32_t x;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(x));
    return x != 0;
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
__device__ __forceinline__ bool h2_not_finite(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// the exponent fields of a pair of f16 (bits 0 … 4 and 16 … 20), 0 for what is not finite
__device__ __forceinline__ uint32_t h2exps(uint32_t w) {
    w &= 0x7fff7fffu;
    return (w & __vcmpltu2(w, 0x7c007c00u)) >> 10 & 0x001f001fu;
}
// four exponents in a word, block b's in the byte where h2exps leaves it: 0, 2, 1, 3
__device__ __forceinline__ constexpr int exp_shift(int b) { return 8 * ((b >> 1) | (b & 1) << 1); }
__device__ __forceinline__ int exp_of(uint32_t bytes, int b) { return (int)((bytes >> exp_shift(b)) & 255u) - KC_EXP; }
// whether any of the `threads` threads at barrier `id` says so
__device__ __forceinline__ bool bar_any(int id, int threads, bool mine) {
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}"
                 : "=r"(any)
                 : "r"((uint32_t)mine), "r"(id), "r"(threads)
                 : "memory");
    return any != 0;
}

// ---- the staging of a tile, by 224 threads: raw rows to registers, later to operands ------------------------------------
// K and V alike: rows of 64 dims (128 bytes, swizzled) in D / 64 halves of 128 keys — K is read along the dims (K-major),
// V along the keys (MN-major), from the same layout. A warp's load covers four whole 128-byte lines; the lanes stand so
// that the eight of a store's phase (one or more keys, units side by side) meet all eight 16-byte pieces of a row.
template <int TYPE, int D>
struct KcRaw {
    static constexpr bool QN = TYPE != KV_F16;
    static constexpr int NB = D / KV_BLOCK, ROW = kv_row_bytes(TYPE, D);
    static constexpr int UPK = ROW / 16;                               // 16-byte units of a key
    static constexpr int UG = TYPE == KV_F16 ? 8 : TYPE == KV_Q8_0 ? 4 : 2;  // units of a key among eight lanes
    static constexpr int PC = 8 / UG;                                  // 16-byte pieces of f16 from a unit
    static constexpr int KPW = 8 / UG * 4 / (D / 64);                  // keys of a warp's load
    static constexpr int STEP = KC_LOADERS * KPW;                      // keys from one unit of a thread to its next
    static constexpr int KU = (KC_KEYS + STEP - 1) / STEP;             // units of a thread, the last one of some warps
    uint4 k[KU], v[KU];
    uint32_t ex[2][QN ? NB / 2 : 1];  // threads 0 … 127: the scales of one key, K's and V's

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
        __device__ __forceinline__ Tile() {}
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
            for (int i = 0; i < KU; i++)
                if (key + i * STEP < KC_KEYS) x[i] = *reinterpret_cast<const uint4*>(p + i * STEP * ROW);
            return;
        }
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int w = t.v0 + key + i * STEP;
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (key + i * STEP < KC_KEYS && w < s.nv) x[i] = *reinterpret_cast<const uint4*>(data + (base + kv_row(c, s.position(w))) * ROW + u * 16);
        }
    }
    __device__ __forceinline__ void load_scales(const KvView& c, const KvSpan& s, size_t base, const Tile& t, int lt) {
        if (QN && lt < KC_KEYS) {
            const int w = t.v0 + lt;
            const bool live = w < s.nv;
            const size_t row = t.run ? t.row + lt : base + (live ? kv_row(c, s.position(w)) : 0);
#pragma unroll
            for (int j = 0; j < NB / 2; j++) {
                ex[0][j] = live ? reinterpret_cast<const uint32_t*>(c.ks + row * NB)[j] : 0u;
                ex[1][j] = live ? reinterpret_cast<const uint32_t*>(c.vs + row * NB)[j] : 0u;
            }
        }
    }
    // The operands, the values of block b times 2^(HEAD - e), e byte b of `exps`. `bad` (an edge tile's V): what is not
    // finite becomes zero and its key is marked.
    __device__ static __forceinline__ void store(const uint4* x, uint8_t* hi, uint8_t* lo, const __half* scale, uint32_t exps,
                                                 uint32_t* bad, int lw, int lane) {
        int key0, u;
        place(lw, lane, key0, u);
        [[maybe_unused]] const float down = exp2i((TYPE == KV_Q8_0 ? 8 : 12) - exp_of(exps, TYPE == KV_Q8_0 ? u >> 1 : u));
#pragma unroll
        for (int i = 0; i < KU; i++) {
            const int key = key0 + i * STEP;
            if (key >= KC_KEYS) break;
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

template <int TYPE, int D, class T, bool LONG>
__global__ void __launch_bounds__(KC_THREADS, 1) k_kv_attn_tc(const __grid_constant__ KvAttnArgs a, int blocks) {
    using P = KcPlan<TYPE, D, T, LONG>;
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
            mbar_init(&sh.pfull[i], 8);
            mbar_init(&sh.odone[i], 1);
        }
        for (int i = 0; i < KC_RING; i++) mbar_init(&sh.xfull[i], 1);
        for (int j = 0; j <= (P::QN ? P::NB : 1); j++) sh.top[0][j] = sh.top[1][j] = 0u;
        mbar_init(&sh.mdone, 1);
        mbar_init(&sh.qfull, 8);
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
    int total = 0, longest = 0;
    if (tid == 0) sh.longest = sh.prefix[0] = 0;
    for (int e0 = 0; e0 < entries; e0 += KC_THREADS) {
        const int e = e0 + tid;
        int sum = 0;
        if (e < entries) {
            int t0, t1;
            rows_of_block(e % blocks, t0, t1);
            KvSpan s;
            s.set(a, e / blocks, t0, t1);
            const int tiles = (s.nv + KC_KEYS - 1) / KC_KEYS;
            longest = max(longest, tiles);
            sum = tiles * c.n_kv;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, sum, o);
            if (lane >= o) sum += y;
        }
        if (lane == 31) sh.wsum[warp] = sum;
        __syncthreads();
        sum += total;
        for (int w = 0; w < KC_THREADS / 32; w++) {
            if (w < warp) sum += sh.wsum[w];
            total += sh.wsum[w];
        }
        if (e < entries) sh.prefix[e + 1] = sum;
        __syncthreads();
    }
    longest = __reduce_max_sync(FULL, longest);
    if (lane == 0 && longest) atomicMax(&sh.longest, longest);
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
    const int least = kv_least_share(total, entries * c.n_kv, 1);
    const int n_cta = min((int)gridDim.x, (total + least - 1) / least);
    const int cta = blockIdx.x;
    KvLine cut;
    cut.cut(total, n_cta);
    int begin, end;
    // Even parts cut most triples in two, and each piece costs the time of some KC_PIECE tiles beside its own (the
    // queries staged, the sums joined); whole ones leave SMs idle. 2214 rows in a window of 512 (280 triples of at most
    // five tiles on 148 SMs): 66 us whole, 121 cut; 666 pairs by 2214 keys twice (96 triples of 8 to 18): 62 and 66; 2048 by
    // 16896 keys four times (256 of 65 to 132): 405 and 272; 8 trees of 61 drafts (128 of 65): 213 and 218.
    kv_share(cut, cta, sh.prefix, entries, c.n_kv, total, sh.longest, (int)gridDim.x, KC_PIECE, KC_PIECE / 2, begin, end);
    KvCursor cc;
    bool any_mma = false;  // (the issuing thread)
    uint32_t qn = 0;
    // a triple: its slot and row block, the keys it sees
    struct Triple {
        int slot, blk, t0, t1;
        KvSpan sp;
        size_t base;
    };
    auto triple = [&](const KvCursor& at) {
        Triple x;
        x.slot = at.b / blocks, x.blk = at.b % blocks;
        rows_of_block(x.blk, x.t0, x.t1);
        x.sp.set(a, x.slot, x.t0, x.t1);
        x.base = kv_index(c, x.slot, at.h, 0);
        return x;
    };
    // the tiles whose every key is seen by every row of the block: at v0 in the sinks, or from `from` to `to`
    struct Plain {
        int ns, from, to;
        __device__ __forceinline__ bool edge(int v0) const { return v0 + KC_KEYS > ns && (v0 < from || v0 > to); }
    };
    auto plain_of = [&](const Triple& x) {
        const KvSpan& sp = x.sp;
        const int shift = sp.ns - sp.lo;  // key = position + shift
        const int lowest = sp.pos + (a.parent ? -1 : x.t0), highest = sp.pos + (a.parent ? sp.m : min(x.t1, sp.m)) - 1;
        // (with a window: past every row's window's start; sinks inside the window's part are left to the mask)
        return Plain{sp.ns, max(sp.ns, c.window ? highest - c.window + 1 + shift : 0), min(sp.nv, lowest + 1 + shift) - KC_KEYS};
    };
    if (warp >= 8 && warp < 15) {
        // ---- the staging: K of tile n + 1, then V of tile n, from the first of the CTA's tiles to the last ----
        const int lw = warp - 8, lt = tid - 256, tiles = end - begin;
        Raw raw{};
        bool ok = true;  // (a thread that gave up still meets the others at every tile's barrier)
        auto find = [&](KvCursor& at, int g) {
            at.at(g, sh.prefix, entries, c.n_kv);
        };
        KvCursor kc;
        Triple kx;
        Plain kp;
        if (tiles > 0) {
            find(kc, begin);
            kx = triple(kc);
            kp = plain_of(kx);
        }
        typename Raw::Tile tv;             // of the V tile to load next: K's of the tile before
        bool next_edge = false, edge = false;
        uint32_t vexp = 0u, kexp = 0u, tops = 0u;  // the exponents in the triple so far: V's blocks', K's; times they moved
        int plain = 0;                     // tiles that follow at 128 rows' distance, whole and seen by every row
        auto load_k = [&](int n) {         // tile n's K and scales; its place is V's next
            if (plain > 0) {
                plain--;
                tv.row += KC_KEYS, tv.v0 += KC_KEYS;
            } else {
                const int g = begin + n;
                if (g >= kc.first + kc.tiles) {
                    find(kc, g);
                    kx = triple(kc);
                    kp = plain_of(kx);
                }
                const KvSpan& sp = kx.sp;
                tv = typename Raw::Tile(c, sp, kx.base, (g - kc.first) * KC_KEYS);
                next_edge = kp.edge(tv.v0);
                if (tv.run && !next_edge && tv.v0 >= sp.ns)
                    plain = min(min((kp.to - tv.v0) / KC_KEYS, (c.n_rows - (int)(tv.row - kx.base)) / KC_KEYS - 1),
                                min(end, kc.first + kc.tiles) - g - 1);
            }
            raw.load_scales(c, kx.sp, kx.base, tv, lt);
            raw.load(raw.k, c.k, c, kx.sp, kx.base, tv, lw, lane);
        };
        auto load_v = [&](int n, const typename Raw::Tile& t, bool e) {
            edge = e;
            if (t.run) {
                raw.load(raw.v, c.v, c, kx.sp, 0, t, lw, lane);
            } else {  // (K may be in the next triple)
                KvCursor at = kc;
                if (begin + n < kc.first) find(at, begin + n);
                const Triple x = triple(at);
                raw.load(raw.v, c.v, c, x.sp, x.base, t, lw, lane);
            }
        };
        // The exponents that the operands are scaled by: one for K (S takes it back with the row's factor), one for each
        // block of 32 dims of V (O is in their units). They stay from tile to tile until a scale passes one, or a triple
        // begins; they are then a power of two above the largest, so that they seldom move.
        auto put_k = [&](int n) {  // → the exponents of V's tile
            const int st = n % NS, x = n % KC_RING;
            if (lt < 4) sh.bad[n % KC_MARKS][lt] = 0u;
            uint32_t kf = 0u, vf = 0u;  // a key's largest exponent of K, those of V's blocks
            if (P::QN && lt < KC_KEYS) {
#pragma unroll
                for (int j = 0; j < P::NB / 2; j++) {
                    reinterpret_cast<uint32_t*>(sh.scale[x][0][lt])[j] = raw.ex[0][j];
                    reinterpret_cast<uint32_t*>(sh.scale[x][1][lt])[j] = raw.ex[1][j];
                    kf = __vmaxu2(kf, h2exps(raw.ex[0][j]));
                    vf |= h2exps(raw.ex[1][j]) << (8 * j);
                }
                kf = max(kf & 0xffffu, kf >> 16);
            }
            if constexpr (P::QN) {
                const bool first = n == 0 || begin + n == kc.first;
                // (bytes below 128: a byte of the difference keeps its top bit unless the exponent is passed)
                const bool pass = first || kf > kexp || (((vexp | 0x80808080u) - vf) & 0x80808080u) != 0x80808080u;
                if (bar_any(2, KC_LOADERS * 32, pass)) {
                    uint32_t* top = sh.top[tops & 1];
                    if (lt < KC_KEYS) {
                        const uint32_t k = __reduce_max_sync(FULL, kf);
                        if (lane == 0) atomicMax(&top[P::NB], k);
#pragma unroll
                        for (int j = 0; j < P::NB; j++) {
                            const uint32_t v = __reduce_max_sync(FULL, vf >> exp_shift(j) & 255u);
                            if (lane == 0) atomicMax(&top[j], v);
                        }
                    }
                    if (lt <= P::NB) sh.top[~tops & 1][lt] = 0u;  // (read before this tile's barrier)
                    bar_sync(2, KC_LOADERS * 32);
                    if (first || top[P::NB] > kexp) kexp = top[P::NB] + 1;
                    uint32_t now = 0u;
#pragma unroll
                    for (int j = 0; j < P::NB; j++) {
                        const uint32_t was = vexp >> exp_shift(j) & 255u;
                        now |= (first || top[j] > was ? top[j] + 1 : was) << exp_shift(j);
                    }
                    vexp = now;
                    tops++;
                }
                if (lt == 0) {
                    sh.exk[x] = exp2i((int)kexp - KC_EXP - P::HEAD), sh.exv[x] = vexp;
                    mbar_arrive(&sh.xfull[x]);
                }
            } else {
                bar_sync(2, KC_LOADERS * 32);
            }
            ok = ok && (n < NS || kc_wait(&sh.kempty[st], (n / NS - 1) & 1, abort_flag, err));
            uint8_t* kh = Kr + st * P::PARTS * P::T_BYTES;
            if (ok) Raw::store(raw.k, kh, kh + P::T_BYTES, sh.scale[x][0][0], kexp * 0x01010101u, nullptr, lw, lane);
            fence_proxy_async();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&sh.kfull[st]);
            return vexp;
        };
        uint32_t eV = 0u;
        // (from -2: one copy of each step's code — the instruction cache is short of room)
#pragma unroll 1
        for (int n = -2; n < tiles; n++) {
            const int st = n % NS, x = n % KC_RING;
            const uint32_t e = eV;
            const typename Raw::Tile t1 = tv;  // of tile n + 1
            const bool e1 = next_edge;
            const bool next = n + 1 >= 0 && n + 1 < tiles;
            if (next) eV = put_k(n + 1);
            if (n + 2 < tiles) load_k(n + 2);
            if (n >= 0) {
                ok = ok && (n < NS || kc_wait(&sh.vempty[st], (n / NS - 1) & 1, abort_flag, err));
                uint8_t* vh = Vr + st * P::PARTS * P::T_BYTES;
                if (ok)
                    Raw::store(raw.v, vh, vh + P::T_BYTES, sh.scale[x][1][0], e, edge ? sh.bad[n % KC_MARKS] : nullptr, lw, lane);
                fence_proxy_async();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&sh.vfull[n & 1]);
            }
            if (next) load_v(n + 1, t1, e1);
        }
    } else if (warp == 15) {
        // ---- the products: Q K^T of tile n + 1, then P V of tile n, the first group's and the second's ----
        // one thread by election, not by its number: the compiler then knows that it is one (10 % of the whole kernel's time)
        if (elect_one()) {
            constexpr uint32_t idS = bg_idesc(KC_KEYS), idO = bg_idesc_mn(D);
            constexpr int HALF = KC_KEYS / 2;
            // the operands' descriptors; a step adds to their address field, in 16-byte units
            const uint64_t qh = bg_desc(smem_u32(Qh)), ql = bg_desc(smem_u32(Ql));
            const uint64_t kd = bg_desc(smem_u32(Kr)), vd = bg_desc_mn(smem_u32(Vr), KC_KEYS * 128);
            constexpr uint64_t T16 = P::T_BYTES / 16;
            auto qk = [&](int n, bool first) -> bool {
                const int st = n % NS;
                // (K first: this wait's own time then passes while the products before are still running)
                if (!kc_wait(&sh.kfull[st], (n / NS) & 1, abort_flag, err)) return false;
                // (a triple's first: its Q is there, and every product of the one before is done)
                if (first ? !kc_wait(&sh.qfull, qn++ & 1, abort_flag, err)
                          // P of tile n - 2 lies over this S: its products are done
                          : n >= 2 && !kc_wait(&sh.odone[n & 1], ((n >> 1) - 1) & 1, abort_flag, err))
                    return false;
                tc_fence_after();
                const uint64_t kh = kd + st * P::PARTS * T16, kl = kh + T16;
                // the small products first: a sum loses what falls below its last bit at every product added
                constexpr int SMALL = (P::LO ? 1 : 0) + (P::QN ? 1 : 0);
#pragma unroll 1
                for (int x = 0; x <= SMALL; x++) {
                    const uint64_t aq = P::LO && x == 0 ? ql : qh, bk = P::QN && x == (P::LO ? 1 : 0) ? kl : kh;
#pragma unroll 1
                    for (int y = 0; y < D / 64; y++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint64_t o = (uint64_t)(y * (128 * 128 / 16) + k * 2);
                            mma_f16(tmem + (n & 1) * KC_KEYS, aq + o, bk + o, idS, x + y + k > 0 ? 1u : 0u);
                        }
                }
                mma_commit(&sh.sfull[n & 1]);
                mma_commit(&sh.kempty[st]);
                any_mma = true;
                return true;
            };
            auto pv = [&](int n, bool fresh) -> bool {
                const int st = n % NS;
                if (!kc_wait(&sh.vfull[n & 1], (n >> 1) & 1, abort_flag, err)) return false;
                if (!kc_wait(&sh.pfull[n & 1], (n >> 1) & 1, abort_flag, err)) return false;
                tc_fence_after();
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const uint64_t vh = vd + st * P::PARTS * T16 + w * HALF * 128 / 16, vl = vh + T16;
                    const uint32_t tP = tmem + (n & 1) * KC_KEYS + w * HALF, tD = tmem + 256 + w * 128;
#pragma unroll
                    for (int k = 0; k < HALF / 16; k++) {  // 32 keys' P: hi in 16 columns, lo in the next 16
                        const uint32_t p = tP + (k >> 1) * 32 + (k & 1) * 8;
                        const uint64_t o = k * 2048 / 16;
                        mma_f16_ts(tD, p, vh + o, idO, (!fresh || k > 0) ? 1u : 0u);
                        if constexpr (P::LO) mma_f16_ts(tD, p + 16, vh + o, idO, 1u);
                        if constexpr (P::QN) mma_f16_ts(tD, p, vl + o, idO, 1u);
                    }
                }
                mma_commit(&sh.odone[n & 1]);
                mma_commit(&sh.vempty[st]);
                return true;
            };
            bool go = true;
            int n = 0;
            for (int seg = begin; seg < end && go;) {
                cc.at(seg, sh.prefix, entries, c.n_kv);
                const int seg_end = min(end, cc.first + cc.tiles), N = seg_end - seg;
#pragma unroll 1
                for (int i = -1; i < N && go; i++) {
                    if (i + 1 < N) go = qk(n + i + 1, i < 0);
                    if (i >= 0) go = go && pv(n + i, P::MOVES ? i % P::FLUSH == 0 : i == 0);
                }
                n += N;
                seg = seg_end;
            }
            if (any_mma) {  // every product complete before the TMEM is given back
                mma_commit(&sh.mdone);
                mbar_wait(&sh.mdone, 0, err);
            }
        }
        __syncwarp();
    } else {
    int n0 = 0;              // tiles of this CTA before the triple
    bool ok = true;          // (a warp that gave up still meets its groups at every barrier)
    for (int seg = begin; seg < end;) {
        cc.at(seg, sh.prefix, entries, c.n_kv);
        const Triple x3 = triple(cc);
        const Plain plain = plain_of(x3);
        const KvSpan& sp = x3.sp;
        const int slot = x3.slot;
        const int seg_end = min(end, cc.first + cc.tiles), N = seg_end - seg;
        const int r0 = x3.blk * KC_M, rows = min(KC_M, sp.m * G - r0);
        if (a.parent && tid < sp.m) sh.parent[tid] = a.parent[(size_t)slot * a.r.T + tid];
        // ---- the queries: hi and lo, a row per warp at a time ----
        {
            constexpr int R = KC_M / 8, V = D / 32;  // a warp's rows; a lane's dims
            alignas(16) T q[R][V];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int r = warp + 8 * i, row = r0 + r;
                const T* qp = static_cast<const T*>(a.q) + slot * a.q_slot + (row / G) * a.q_row +
                              (cc.h * G + row % G) * a.q_head + lane * V;
                using Word = typename KcWord<V * sizeof(T)>::type;
                Word w = {};
                if (r < rows) w = *reinterpret_cast<const Word*>(qp);
                *reinterpret_cast<Word*>(q[i]) = w;
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int r = warp + 8 * i;
                float x[V];
                float f = a.scale * LOG2E;
#pragma unroll
                for (int j = 0; j < V; j++) x[j] = (float)q[i][j];
                if constexpr (P::LO) {  // the row's largest to 2^10 … 2^11
                    float big = 0.0f;
#pragma unroll
                    for (int j = 0; j < V; j++) big = fmaxf(big, fabsf(x[j]));
                    // (of floats that are not negative, the bits' order is theirs)
                    big = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(big)));
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
                    const uint32_t h = P::LO && !P::QN ? pack2_below(x[2 * j], x[2 * j + 1]) : pack2(x[2 * j], x[2 * j + 1]);
                    *reinterpret_cast<uint32_t*>(Qh + at + 4 * j) = h;
                    if constexpr (P::LO) *reinterpret_cast<uint32_t*>(Ql + at + 4 * j) = rest2(x[2 * j], x[2 * j + 1], h);
                }
            }
            fence_proxy_async();
            tc_fence_before();  // (the last triple's sums are read)
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.qfull);
        }
        bar_sync(3, 256);
        if (a.parent) {
            if (tid < sp.m) sh.depth[tid] = kv_depth(tid, sh.parent, err);
            bar_sync(3, 256);
        }
        {
            // ---- the rows: thread r of group wg owns pair r0 + r (TMEM lane r), keys 64 wg … 64 wg + 63 of every tile ----
            const int wg = warp >> 2, r = tid & 127;
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t tO = tmem + lanes + 256 + wg * 128;
            const int row = min((r0 + r) / G, sp.m - 1);
            KvSight sight;
            if (a.parent)
                kv_draft(c, sp, row, sh.parent, sh.depth, sight);
            else
                sight.rows(c, sp, sp.pos + row, sp.pos + row);
            const float fac0 = sh.fac[r];
            float m = -INFINITY, l = 0.0f;
            uint32_t vexp = 0u;  // the exponents of the blocks of O
            // block b's factor from O's unit
            auto unit = [&](int b) { return P::QN ? exp2i(exp_of(vexp, b) - P::HEAD) : 1.0f; };
            // the group's sums in memory, [D][128]: their reference
            float m_kept = -INFINITY;
            float* kept = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + KV_TICKETS) +
                          (size_t)gridDim.x * 2 * P::PART + (size_t)(2 * cta + wg) * D * KC_M + r;
            constexpr int HALF = KC_KEYS / 2;
            // an edge tile's values that are not finite were taken out of the product (a row that does not see them must not
            // meet them as 0 times infinity); a row that sees one is spoilt as a whole
            auto marks = [&](int i) {
                const int v0 = (seg - cc.first + i) * KC_KEYS;
                if (!plain.edge(v0)) return;
#pragma unroll
                for (int ch = 0; ch < 2; ch++) {
                    const uint32_t bad = sh.bad[(n0 + i) % KC_MARKS][2 * wg + ch];
                    if (bad && (bad & sight.mask(v0 + HALF * wg + 32 * ch))) l = NAN;
                }
            };
            auto tile = [&](int i) -> bool {  // the weights of tile i; false: a wait gave up
                const int n = n0 + i, x = n % KC_RING, v0 = (seg - cc.first + i) * KC_KEYS;
                const uint32_t tS = tmem + lanes + (n & 1) * KC_KEYS + wg * HALF;
                const bool edge = plain.edge(v0);
                float fac = fac0;
                uint32_t ve = 0u;
                if constexpr (P::QN) {
                    if (!kc_wait_warp(&sh.xfull[x], (n / KC_RING) & 1, abort_flag, err)) return false;
                    fac *= sh.exk[x];
                    ve = sh.exv[x];
                }
                if (!kc_wait_warp(&sh.sfull[n & 1], (n >> 1) & 1, abort_flag, err)) return false;
                tc_fence_after();
                if (i >= 2) marks(i - 2);  // (S of this tile says that V of that one was used)
                uint32_t s[HALF];
                tmem_ld32(tS, s);
                tmem_ld32(tS + 32, s + 32);
                tmem_wait_ld();
                if (edge) {  // what the row does not see is taken out
#pragma unroll
                    for (int ch = 0; ch < 2; ch++) {
                        const uint32_t see = sight.mask(v0 + HALF * wg + 32 * ch);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!((see >> j) & 1)) s[32 * ch + j] = 0xff800000u;
                    }
                }
                float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < HALF; j++) mq[j & 3] = fmaxf(mq[j & 3], __uint_as_float(s[j]));
                const float mt = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * fac;
                const bool flush = P::MOVES && i > 0 && i % P::FLUSH == 0;
                const float m_was = m;
                if (i == 0) {
                    m = mt;
                } else if (flush) {  // (O starts afresh)
                    m = fmaxf(m, mt);
                    if (m_was != -INFINITY) l *= ex2(m_was - m);
                } else if (__any_sync(FULL, mt > m + KC_LAG || (P::QN && ve != vexp))) {
                    // (the reference moves, or a block's exponent did. Warp-uniform: TMEM loads and stores are the whole
                    // warp's; a row that stays scales by 1)
                    if (!kc_wait_warp(&sh.odone[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, err)) return false;
                    tc_fence_after();
                    const bool up = mt > m + KC_LAG;
                    const float f = up ? ex2(m - mt) : 1.0f;
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t o[16];
                        const float g = P::QN ? f * exp2i(exp_of(vexp, d >> 5) - exp_of(ve, d >> 5)) : f;
                        tmem_ld16(tO + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * g);
                        tmem_st16(tO + d, o);
                    }
                    l *= f;
                    if (up) m = mt;
                }
                const float ref = KC_BIAS - (m == -INFINITY ? 0.0f : m);
                float sum[2] = {0.0f, 0.0f};
#pragma unroll
                for (int ch = 0; ch < 2; ch++) {
                    uint32_t h[16], lo[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float p0 = ex2(fmaf(__uint_as_float(s[32 * ch + 2 * j]), fac, ref));
                        const float p1 = ex2(fmaf(__uint_as_float(s[32 * ch + 2 * j + 1]), fac, ref));
                        sum[0] += p0, sum[1] += p1;
                        h[j] = pack2(p0, p1);
                        if constexpr (P::LO) lo[j] = rest2(p0, p1, h[j]);
                    }
                    tmem_st16(tS + 32 * ch, h);
                    if constexpr (P::LO) tmem_st16(tS + 32 * ch + 16, lo);
                }
                l += sum[0] + sum[1];
                tmem_wait_st();
                if (flush) {
                    if (!kc_wait_warp(&sh.odone[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, err)) return false;
                    tc_fence_after();
                    const float f = m_kept == -INFINITY ? 0.0f : ex2(m_kept - m_was);
                    const bool more = i > P::FLUSH;
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        uint32_t o[32];
                        float k[32];
                        const float g = unit(d >> 5);
                        tmem_ld32(tO + d, o);
#pragma unroll
                        for (int j = 0; j < 32; j++) k[j] = more ? __ldcg(&kept[(d + j) * KC_M]) : 0.0f;
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j++) __stcg(&kept[(d + j) * KC_M], fmaf(k[j], f, __uint_as_float(o[j]) * g));
                    }
                    m_kept = m_was;
                }
                vexp = ve;
                return true;
            };
            for (int i = 0; i < N; i++) {
                const int n = n0 + i;
                ok = ok && tile(i);
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&sh.pfull[n & 1]);
            }
            // both groups' products are done
            const int last = n0 + N - 1;
            ok = __all_sync(FULL, ok && *abort_flag == 0);
            ok = ok && kc_wait_warp(&sh.odone[last & 1], (last >> 1) & 1, abort_flag, err);
            if (N > 1) marks(N - 2);
            marks(N - 1);
            sh.ml[wg][0][r] = m;
            sh.ml[wg][1][r] = l;
            sh.ml[wg][2][r] = m_kept == -INFINITY ? 0.0f : ex2(m_kept - m);
            tc_fence_after();
            bar_sync(3, 256);
            // the row's sums: each group writes half of the dims
            const float ma = sh.ml[0][0][r], mb = sh.ml[1][0][r];
            const float mx = fmaxf(ma, mb), safe = mx == -INFINITY ? 0.0f : mx;
            const float fa = ex2(ma - safe), fb = ex2(mb - safe);
            const float lt = sh.ml[0][1][r] * fa + sh.ml[1][1][r] * fb;
            const bool whole = N == cc.tiles;
            const int c0 = whole ? 0 : cut.owner(cc.first);
            float* mine = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + KV_TICKETS) +
                          (size_t)(2 * cta + (cta == c0)) * P::PART;
            const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
            // (Q's memory is free: every product is done) the rows of the output, 16-byte pieces moved among eight
            constexpr int ROW = D * sizeof(T), E = 16 / sizeof(T);  // E elements of a piece
            auto stage = [&](int r, int d, const float* y) {  // dims d … d + 15 of row r
#pragma unroll
                for (int j = 0; j < 16 / E; j++) {
                    uint4 w;
                    if constexpr (P::LO)
                        w = make_uint4(__float_as_uint(y[4 * j]), __float_as_uint(y[4 * j + 1]), __float_as_uint(y[4 * j + 2]),
                                       __float_as_uint(y[4 * j + 3]));
                    else
                        w = make_uint4(pack2(y[8 * j], y[8 * j + 1]), pack2(y[8 * j + 2], y[8 * j + 3]),
                                       pack2(y[8 * j + 4], y[8 * j + 5]), pack2(y[8 * j + 6], y[8 * j + 7]));
                    *reinterpret_cast<uint4*>(Qh + r * ROW + (((d / E + j) ^ (r & 7)) << 4)) = w;
                }
            };
            bool emit = whole && ok;
            if (ok) {
#pragma unroll 1
                for (int d = wg * (D / 2); d < (wg + 1) * (D / 2); d += 16) {
                    uint32_t o[16], o2[16];
                    const float oa = fa * unit(d >> 5), ob = fb * unit(d >> 5);
                    tmem_ld16(tmem + lanes + 256 + d, o);
                    tmem_ld16(tmem + lanes + 384 + d, o2);
                    float y[16] = {};
                    if (P::MOVES && N > P::FLUSH) {
                        const float *k0 = kept - wg * D * KC_M, *k1 = k0 + D * KC_M;
                        const float ga = fa * sh.ml[0][2][r], gb = fb * sh.ml[1][2][r];
#pragma unroll
                        for (int j = 0; j < 16; j++) y[j] = fmaf(__ldcg(&k1[(d + j) * KC_M]), gb, __ldcg(&k0[(d + j) * KC_M]) * ga);
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j++) y[j] = fmaf(__uint_as_float(o2[j]), ob, fmaf(__uint_as_float(o[j]), oa, y[j]));
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 16; j++) y[j] = lt == 0.0f ? 0.0f : y[j] * inv;
                        stage(r, d, y);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) __stcg(&mine[(d + j) * KC_M + r], y[j]);
                    }
                }
                if (!whole && wg == 0) {
                    __stcg(&mine[D * KC_M + r], mx);
                    __stcg(&mine[(D + 1) * KC_M + r], lt);
                }
                if (!whole) __threadfence();
            }
            tc_fence_before();
            bar_sync(3, 256);
            // ---- a triple that lies in several CTAs: the last of them joins the parts in the CTAs' order ----
            if (!whole) {
                const int c1 = cut.owner(cc.first + cc.tiles - 1);
                uint32_t* tickets = static_cast<uint32_t*>(a.work);
                if (tid == 0) {  // (after a wait that gave up nothing is joined; the host sets the tickets back)
                    const bool last_one = *abort_flag == 0 && atomicAdd(&tickets[c0], 1u) == (uint32_t)(c1 - c0);
                    if (last_one) tickets[c0] = 0;
                    __threadfence();
                    sh.last = last_one;
                }
                bar_sync(3, 256);
                emit = sh.last;
                if (emit) {
                    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.work) + KV_TICKETS);
                    auto of = [&](int i) { return parts + (size_t)(2 * i + (i == c0)) * P::PART; };
                    // (row, dim) pairs of the rows in use, a warp's side by side; each thread's several in flight at once
                    const int R = (rows + 31) & ~31;
#pragma unroll 1
                    for (int e0 = tid; e0 < R * (D / 16); e0 += 256) {
                        const int rr = e0 % R, d = e0 / R * 16;
                        float top = -INFINITY, sum = 0.0f, y[16] = {};
#pragma unroll 8
                        for (int i = c0; i <= c1; i++) top = fmaxf(top, __ldcg(&of(i)[D * KC_M + rr]));
                        if (top == -INFINITY) top = 0.0f;
#pragma unroll 2
                        for (int i = c0; i <= c1; i++) {
                            const float* q = of(i);
                            const float f = ex2(__ldcg(&q[D * KC_M + rr]) - top);
                            sum = fmaf(__ldcg(&q[(D + 1) * KC_M + rr]), f, sum);
#pragma unroll
                            for (int j = 0; j < 16; j++) y[j] = fmaf(__ldcg(&q[(d + j) * KC_M + rr]), f, y[j]);
                        }
                        const float scale = 1.0f / sum;
#pragma unroll
                        for (int j = 0; j < 16; j++) y[j] = sum == 0.0f ? 0.0f : y[j] * scale;
                        stage(rr, d, y);
                    }
                }
                bar_sync(3, 256);
            }
            if (emit) {
                constexpr int PC = ROW / 16;
                for (int e = tid; e < rows * PC; e += 256) {
                    const int rr = e / PC, pc = e % PC;
                    T* op = static_cast<T*>(a.out) + slot * a.o_slot + ((r0 + rr) / G) * a.o_row + (cc.h * G + (r0 + rr) % G) * a.o_head;
                    reinterpret_cast<uint4*>(op)[pc] = *reinterpret_cast<const uint4*>(Qh + rr * ROW + ((pc ^ (rr & 7)) << 4));
                }
            }
            bar_sync(3, 256);
        }
        n0 += N;
        seg = seg_end;
    }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int TYPE, int D, class T, bool LONG>
static cudaError_t launch_tc(cudaStream_t st, const KvAttnArgs& a, int blocks, bool pdl) {
    using P = KcPlan<TYPE, D, T, LONG>;
    static PerDeviceOnce once;
    once([] { cudaFuncSetAttribute(k_kv_attn_tc<TYPE, D, T, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::SMEM); });
    return kv_launch(k_kv_attn_tc<TYPE, D, T, LONG>, dim3(a.num_sms), KC_THREADS, P::SMEM, st, pdl, a, blocks);
}
// the most keys that a row can see
static long keys_of(const KvAttnArgs& a) {
    return a.c.window ? min((long)a.c.n_rows, (long)a.c.window + a.c.sinks + a.r.T) : a.c.n_rows;
}
// f16 rows: keys from which sums are moved out of TMEM (1024 products to a sum: they may lose 10^-4 of it, two fifths of the
// output's rounding). It takes code that all calls would pay for: 4 x 512 rows by 16.9k f16 keys 273 us, with it 301.
static bool is_long(const KvAttnArgs& a) { return keys_of(a) > (a.c.type == KV_F16 ? 32768 : 16384); }
template <int TYPE, int D>
static cudaError_t launch_rows(cudaStream_t st, const KvAttnArgs& a, int blocks, bool pdl) {
    if (!a.half) return launch_tc<TYPE, D, float, false>(st, a, blocks, pdl);
    return is_long(a) ? launch_tc<TYPE, D, __half, true>(st, a, blocks, pdl) : launch_tc<TYPE, D, __half, false>(st, a, blocks, pdl);
}
template <int TYPE>
static cudaError_t launch_type(cudaStream_t st, const KvAttnArgs& a, int blocks, bool pdl) {
    return a.c.d == 128 ? launch_rows<TYPE, 128>(st, a, blocks, pdl) : launch_rows<TYPE, 64>(st, a, blocks, pdl);
}
// tickets, two parts for each CTA, the groups' sums (of heads of 128)
size_t kv_attention_many_work(int num_sms) { return KV_TICKETS + (size_t)num_sms * 2 * ((128 + 2) + 128) * KC_M * 4; }
// (row, query head) pairs of a kv head in one slot that one call takes
long kv_attention_many_rows() { return (long)KV_LINE * KC_M; }
static int blocks_of(const KvAttnArgs& a) { return (int)(((long)a.r.T * (a.n_head / a.c.n_kv) + KC_M - 1) / KC_M); }
// slots of one launch: their (slot, row block) pairs have places in the line, and its tiles are counted in 32 bits (0: not
// even one slot's)
int kv_attention_many_slots(const KvAttnArgs& a) {
    const KvView& c = a.c;
    const int blocks = blocks_of(a);
    const long tiles = (keys_of(a) + KC_KEYS - 1) / KC_KEYS * c.n_kv * blocks;
    return (int)min((long)(KV_LINE / blocks), 0x7fffffffL / tiles);
}
cudaError_t launch_kv_attention_many(cudaStream_t st, const KvAttnArgs& all, bool pdl) {
    const int blocks = blocks_of(all), slots = kv_attention_many_slots(all);
    for (int b = 0; b < all.c.n_slot; b += slots) {
        const KvAttnArgs a = kv_slots(all, b, min(slots, all.c.n_slot - b));
        const cudaError_t e = a.c.type == KV_F16    ? launch_type<KV_F16>(st, a, blocks, pdl)
                              : a.c.type == KV_Q8_0 ? launch_type<KV_Q8_0>(st, a, blocks, pdl)
                                                    : launch_type<KV_Q4_0>(st, a, blocks, pdl);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace ocr
