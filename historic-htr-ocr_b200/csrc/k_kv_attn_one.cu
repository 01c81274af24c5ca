// k_kv_attn_one.cu — attention of one or two (row, query head) pairs per kv head over a q8_0 or q4_0 cache: the decode
// step. Formula, line of tiles, rings and joins are k_kv_attn.cu's; the products are whole numbers.
//
// Bound: memory, if the instructions fit beside it: a key of 128 dims is 272 bytes in q8_0, so an SM gets 32 of them in
// about 380 cycles, and turning their quants into f16 alone takes longer than that. So the quants stay what they are:
// int8 operands of m16n8k32 (s8 x s8 → s32, the same 8 cycles as the f16 product of half its depth).
//   S: the query becomes four signed digits to base 256 of a whole number q 2^k (its largest value just below 2^29), a
//      digit to a column: rows 0, 1 in columns 0, 1 (lowest digit), … 6, 7 (highest). Each block of 32 dims is one
//      product; its exact sums, times the key's block scale, add up in f32; a row's four columns are added.
//   O: a weight times its value's block scale, p d 2^(29 - e) (e from the tile's largest scale; p <= 1), becomes a whole
//      number, and its bytes the digits, again a column each. V is the other operand, four keys' bytes to a word (a
//      4 x 4 transposition by byte permutes).
// A q4_0 nibble n becomes the byte 16 (n - 8) by a shift and one logic operation. The accumulators start at the bits of
// 1.5 2^23, so a sum comes out as a float less a constant (|sums| stay below 2^22: 32 products of 7 bits each, at most
// two of those). Rounding: 2^-30 of a row's largest query value, 2^-30 of the tile's largest scale (on weights whose
// largest is 1), and 2^-24 of each. (Three digits of 21 bits: errors of 2 to 6 10^-6 of the output, three times the
// f32 formula's own.)
// Measured: 32 slots of some 3100 keys, 8 kv heads, two query heads each, q8_0: 55 us, 3.9 TB/s (60 % of a copy's rate; issue
// 52 % busy, ALU 35, loads and stores 28: the digits' packing and the joins, no single unit); the same in a q4_0 ring of 1028
// keys 25 us; one slot of 2304 keys 13 us, latency.
#include "kv_tile.cuh"

namespace ocr {

constexpr int KO_WARPS = 12, KO_THREADS = KO_WARPS * 32;
constexpr int KO_ROWS = 2;
constexpr int KO_MAGIC = 0x4B400000;       // 1.5 2^23
constexpr float KO_MAGIC_F = 12582912.0f;
constexpr float KO_DIGITS = 8421504.0f;    // 0x808080: half a digit in each of the three lower places: signed digits

__device__ __forceinline__ void mma16832(int* d, const uint32_t* a, uint32_t b0, uint32_t b1, const int* c) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// the low or the high nibbles of four bytes as 16 (n - 8)
__device__ __forceinline__ uint32_t nibbles_s8(uint32_t w, bool high) {
    return ((high ? w : w << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
}
__device__ __forceinline__ uint32_t h2max_nan(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float half_of(uint32_t w, int i) {
    return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffffu)));
}

template <int TYPE, int D, class T>
__global__ void __launch_bounds__(KO_THREADS, 1) k_kv_attn_one(const __grid_constant__ KvAttnArgs a) {
    using KT = KaTile<TYPE, D>;
    using Stream = KaStream<TYPE, D, 1, KO_WARPS>;
    constexpr int KEYS = KT::KEYS, MT = KEYS / 16, NB = KT::NB, NH = NB / 2, STAGES = Stream::STAGES;
    constexpr float Q4 = TYPE == KV_Q4_0 ? 1.0f / 16 : 1.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ KaLine line;
    __shared__ KvSight s_sight[KO_ROWS];
    __shared__ int s_parent[KO_ROWS], s_depth[KO_ROWS];
    __shared__ float s_ml[2][KO_ROWS][KO_WARPS];
    __shared__ int s_last;
    pdl_trigger();
    pdl_wait();
    const KvView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int G = a.n_head / c.n_kv;
    const int total = kv_line_sums<KEYS, D, T, KO_THREADS>(a, line);
    const int share = kv_least_share(total, c.n_slot * c.n_kv, KO_WARPS);
    const int n_cta = min((int)gridDim.x, (total + share - 1) / share), cta = blockIdx.x;
    KvLine cut;
    cut.cut(total, n_cta);
    int begin, end;
    kv_share(cut, cta, line.prefix, c.n_slot, c.n_kv, total, line.longest, (int)gridDim.x, KA_PIECE, KA_PIECE, begin, end);
    if (begin >= end) return;
    uint8_t* ring = smem + warp * KA_RING;
    float* joined = reinterpret_cast<float*>(smem + KO_WARPS * KA_RING);  // [warp][row][dim]
    Stream stream(a, line, begin, end, warp, lane, ring);
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) stream.load();

    // column g's digit and row: that byte of four whole numbers, the lower three digits 128 less
    const int digit = g >> 1, grow = g & 1;
    const uint32_t sel = (uint32_t)digit * 0x11u + 0x40u, flip = digit == 3 ? 0u : 0x80808080u;
    auto pick = [&](int x0, int x1, int x2, int x3) {
        return __byte_perm(__byte_perm(x0, x1, sel), __byte_perm(x2, x3, sel), 0x5410) ^ flip;
    };
    const float place = __uint_as_float((uint32_t)(127 + 8 * t) << 23);  // 256^t, of this lane's columns 2t, 2t + 1
    const int zero[4] = {KO_MAGIC, KO_MAGIC, KO_MAGIC, KO_MAGIC};
    // where the lane reads its keys: S takes rows g, g + 8 of 16 keys (keys kA and kA + 2), V keys 4t … 4t + 3
    const int kA = 4 * (g >> 1) + (g & 1);

    int done = 0, ct = begin + warp;
    for (int seg = begin; seg < end;) {
        KvCursor cc;
        KvSpan sp;
        cc.at(seg, line.prefix, c.n_slot, c.n_kv);
        sp.set(a, line.pos[cc.b], line.m[cc.b], 0, a.r.T);
        const int seg_end = min(end, cc.first + cc.tiles), rows = sp.m * G;
        const bool many = a.r.T > 1 || a.parent;  // (else every row sees the whole span)
        if (many) {
            if (a.parent) {
                if (tid < sp.m) s_parent[tid] = a.parent[(size_t)cc.b * a.r.T + tid];
                __syncthreads();
                if (tid < sp.m) s_depth[tid] = kv_depth(tid, s_parent, a.err);
                __syncthreads();
            }
            if (tid < KO_ROWS) {
                const int row = min(tid / G, sp.m - 1);
                if (a.parent)
                    kv_draft(c, sp, row, s_parent, s_depth, s_sight[tid]);
                else
                    s_sight[tid].rows(c, sp, sp.pos + row, sp.pos + row);
            }
            __syncthreads();
        }
        // ---- the query's digits: column g is digit `digit` of row `grow` ----
        uint32_t qd[NB][2];
        float sfac[2];  // of columns 2t, 2t + 1
        {
            const bool live = grow < rows;
            const T* qp = static_cast<const T*>(a.q) + cc.b * a.q_slot + (grow / G) * a.q_row + (cc.h * G + grow % G) * a.q_head;
            float x[NB][8];  // the lane's dims of each block, as K's words hold them
            float big = 0.0f;  // (infinite where a value is an infinity or a NaN)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int d = 32 * b + (TYPE == KV_Q8_0 ? 8 * t + i : 4 * t + (i & 3) + 16 * (i >> 2));
                    x[b][i] = live ? (float)qp[d] : 0.0f;
                    big = fmaxf(big, fabsf(x[b][i]) <= 3.4028234e38f ? fabsf(x[b][i]) : INFINITY);
                }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) big = fmaxf(big, __shfl_xor_sync(FULL, big, o));
            const bool fine = big <= 3.4028234e38f;
            // 2^(e - 1) <= big < 2^e: times 2^(29 - e)
            const int e = big > 0.0f && fine ? max(-100, (int)(__float_as_uint(big) >> 23) - 126) : 0;
            const float up = __uint_as_float((uint32_t)(127 + min(29 - e, 120)) << 23);
            const float down = __uint_as_float((uint32_t)(127 - min(29 - e, 120)) << 23);
            // (a query that is not finite makes its scores NaN)
            const float f = fine ? a.scale * LOG2E * Q4 * down : NAN;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    int n[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) n[i] = __float2int_rn(fmaf(fine ? x[b][4 * u + i] : 0.0f, up, KO_DIGITS));
                    qd[b][u] = pick(n[0], n[1], n[2], n[3]);
                }
            sfac[0] = __shfl_sync(FULL, f, 0) * place;   // row 0 is column 0's
            sfac[1] = __shfl_sync(FULL, f, 4) * place;
        }
        float o[D / 16][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        auto compute = [&](int tile, const uint8_t* st, auto edge_) {
            constexpr bool EDGE = decltype(edge_)::value;
            const uint8_t *kt = st, *vt = st + KT::K_BYTES, *kst = st + 2 * KT::K_BYTES, *vst = kst + KT::S_BYTES;
            const int v0 = (tile - cc.first) * KEYS;
            // ---- S ----
            float p[MT][4];
#pragma unroll
            for (int i = 0; i < MT; i++) {
                __half2 dk[2][NH];
                load_scales<NB>(dk[0], kst, 16 * i + kA), load_scales<NB>(dk[1], kst, 16 * i + kA + 2);
#pragma unroll
                for (int j = 0; j < 4; j++) p[i][j] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t ka[4];
                    if constexpr (TYPE == KV_Q8_0) {
                        const uint2 A = *reinterpret_cast<const uint2*>(kt + KT::off(16 * i + kA, 2 * b + (t >> 1), false) + (t & 1) * 8);
                        const uint2 B = *reinterpret_cast<const uint2*>(kt + KT::off(16 * i + kA + 2, 2 * b + (t >> 1), false) + (t & 1) * 8);
                        ka[0] = A.x, ka[1] = B.x, ka[2] = A.y, ka[3] = B.y;
                    } else {
                        const uint32_t A = *reinterpret_cast<const uint32_t*>(kt + KT::off(16 * i + kA, b, false) + t * 4);
                        const uint32_t B = *reinterpret_cast<const uint32_t*>(kt + KT::off(16 * i + kA + 2, b, false) + t * 4);
                        ka[0] = nibbles_s8(A, false), ka[1] = nibbles_s8(B, false), ka[2] = nibbles_s8(A, true), ka[3] = nibbles_s8(B, true);
                    }
                    int acc[4];
                    mma16832(acc, ka, qd[b][0], qd[b][1], zero);
                    const float dA = b & 1 ? __high2float(dk[0][b / 2]) : __low2float(dk[0][b / 2]);
                    const float dB = b & 1 ? __high2float(dk[1][b / 2]) : __low2float(dk[1][b / 2]);
#pragma unroll
                    for (int j = 0; j < 4; j++) p[i][j] = fmaf(__int_as_float(acc[j]) - KO_MAGIC_F, j < 2 ? dA : dB, p[i][j]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {  // the digits' columns: 2t, 2t + 1 of t = 0 … 3
                    p[i][j] *= sfac[j & 1];
                    p[i][j] += __shfl_xor_sync(FULL, p[i][j], 1);
                    p[i][j] += __shfl_xor_sync(FULL, p[i][j], 2);
                }
            }
            uint64_t col_seen = 0;
            if constexpr (EDGE) {
                auto sees = [&](int row, int v) {
                    const int left = sp.nv - v;
                    return many ? s_sight[row].mask(v) : left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
                };
                uint32_t mask[2][(KEYS + 31) / 32];
#pragma unroll
                for (int w = 0; w < (KEYS + 31) / 32; w++) {
                    mask[0][w] = sees(0, v0 + 32 * w), mask[1][w] = sees(1, v0 + 32 * w);
                    col_seen |= (uint64_t)(grow ? mask[1][w] : mask[0][w]) << (32 * w);
                }
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (!((mask[j & 1][i / 2] >> ((16 * i + kA + 2 * (j >> 1)) & 31)) & 1)) p[i][j] = -INFINITY;
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
                const float mn = fmaxf(m[j], x);
                ref[j] = mn == -INFINITY ? 0.0f : mn;
                alpha[j] = ex2(m[j] - ref[j]);
                m[j] = mn;
            }
            if (__any_sync(FULL, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int d = 0; d < D / 16; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[d][j] *= alpha[j & 1];
                l[0] *= alpha[0], l[1] *= alpha[1];
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    p[i][j] = ex2(p[i][j] - ref[j & 1]);
                    l[j & 1] += p[i][j];
                }
            // ---- the weights of column g's row for keys 16 i + 4t … 4t + 3: row r of S is held by lanes of g = r % 8, row
            //      `grow` of P by those of t = 2 grow ----
            float w[MT][4];
            const int from = 8 * t + 2 * grow;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float x = t >= 2 ? p[i][2 * u + 1] : p[i][2 * u];
                    w[i][2 * u] = __shfl_sync(FULL, x, from);
                    w[i][2 * u + 1] = __shfl_sync(FULL, x, from + 4);
                }
            // ---- the values' scales, and the tile's largest of each block ----
            __half2 dv[MT][4][NH];
            uint32_t top[NH];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    load_scales<NB>(dv[i][u], vst, 16 * i + 4 * t + u);
                    if (EDGE && !((col_seen >> (16 * i + 4 * t + u)) & 1))  // (0 times a scale that is no number is not 0)
#pragma unroll
                        for (int b = 0; b < NH; b++) dv[i][u][b] = __float2half2_rn(0.0f);
#pragma unroll
                    for (int b = 0; b < NH; b++) {
                        const uint32_t x = *reinterpret_cast<const uint32_t*>(&dv[i][u][b]) & 0x7fff7fffu;
                        top[b] = i + u == 0 ? x : h2max_nan(top[b], x);
                    }
                }
            bool bad = false;
#pragma unroll
            for (int b = 0; b < NH; b++) {
                top[b] = h2max_nan(top[b], __shfl_xor_sync(FULL, top[b], 1));
                top[b] = h2max_nan(top[b], __shfl_xor_sync(FULL, top[b], 2));
                bad |= (top[b] & 0xffffu) >= 0x7c00u || (top[b] >> 16) >= 0x7c00u;
            }
            const uint32_t spoilt = __ballot_sync(FULL, bad);  // columns 0 and 1 are rows 0 and 1
            if (spoilt) {
                if (spoilt & 0xfu) l[0] = NAN;
                if (spoilt & 0xf0u) l[1] = NAN;
            }
            // ---- O += V^T P ----
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float big = half_of(top[b / 2], b & 1);
                // 2^(e - 1) <= big < 2^e: p d 2^(29 - e) < 2^29
                const int e = big > 0.0f ? min(17, (int)(__float_as_uint(big) >> 23) - 126) : 0;
                const float down = __uint_as_float((uint32_t)(127 + 29 - e) << 23);
                float up[2];  // of columns 2t, 2t + 1 (the rows may see different keys)
                up[0] = up[1] = __uint_as_float((uint32_t)(127 - 29 + e) << 23);
                if (EDGE && many) up[0] = __shfl_sync(FULL, up[0], 0), up[1] = __shfl_sync(FULL, up[1], 4);
                up[0] *= place * Q4, up[1] *= place * Q4;
                int acc[2][4];
#pragma unroll
                for (int k = 0; k < MT / 2; k++) {  // 32 keys: 16 i + 4t … of i = 2k, then of 2k + 1
                    uint32_t pd[2], va[2][4];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int i = 2 * k + u;
                        int n[4];
                        uint32_t x[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float d = b & 1 ? __high2float(dv[i][j][b / 2]) : __low2float(dv[i][j][b / 2]);
                            n[j] = __float2int_rn(fmaf(w[i][j], d * down, KO_DIGITS));
                        }
                        pd[u] = pick(n[0], n[1], n[2], n[3]);
                        if constexpr (TYPE == KV_Q8_0) {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                x[j] = *reinterpret_cast<const uint32_t*>(vt + KT::off(16 * i + 4 * t + j, 2 * b + (g >> 2), true) + (g & 3) * 4);
                            // words of one dim's four keys: dims 4g … 4g + 3 of the block
                            const uint32_t y0 = __byte_perm(x[0], x[1], 0x5140), y1 = __byte_perm(x[0], x[1], 0x7362);
                            const uint32_t y2 = __byte_perm(x[2], x[3], 0x5140), y3 = __byte_perm(x[2], x[3], 0x7362);
                            va[0][2 * u] = __byte_perm(y0, y2, 0x5410), va[0][2 * u + 1] = __byte_perm(y0, y2, 0x7632);
                            va[1][2 * u] = __byte_perm(y1, y3, 0x5410), va[1][2 * u + 1] = __byte_perm(y1, y3, 0x7632);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                x[j] = *reinterpret_cast<const uint16_t*>(vt + KT::off(16 * i + 4 * t + j, b, true) + g * 2);
                            const uint32_t y0 = __byte_perm(x[0], x[1], 0x5410), y1 = __byte_perm(x[2], x[3], 0x5410);
                            const uint32_t z0 = __byte_perm(y0, y1, 0x6420), z1 = __byte_perm(y0, y1, 0x7531);
                            // dims 2g, 2g + 1 (low nibbles) and 16 + 2g, 17 + 2g (high)
                            va[0][2 * u] = nibbles_s8(z0, false), va[0][2 * u + 1] = nibbles_s8(z1, false);
                            va[1][2 * u] = nibbles_s8(z0, true), va[1][2 * u + 1] = nibbles_s8(z1, true);
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 2; s++) mma16832(acc[s], va[s], pd[0], pd[1], k ? acc[s] : zero);
                }
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[2 * b + s][j] = fmaf(__int_as_float(acc[s][j]) - KO_MAGIC_F, up[j & 1], o[2 * b + s][j]);
            }
        };

        for (; ct < seg_end; ct += KO_WARPS, done++) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            stream.load();  // into the stage that was computed last
            const uint8_t* st = ring + done % STAGES * KT::STAGE;
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

        // ---- the warps' parts side by side: dims of tile d's rows g and g + 8 ----
        auto dim = [&](int d, int up) {
            return TYPE == KV_Q8_0 ? 32 * (d >> 1) + 4 * g + 2 * (d & 1) + up : 32 * (d >> 1) + 16 * (d & 1) + 2 * g + up;
        };
#pragma unroll
        for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[d][j] += __shfl_xor_sync(FULL, o[d][j], 1);
                o[d][j] += __shfl_xor_sync(FULL, o[d][j], 2);
                if (t == (d & 3)) joined[(warp * KO_ROWS + (j & 1)) * D + dim(d, j >> 1)] = o[d][j];
            }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            l[j] += __shfl_xor_sync(FULL, l[j], 4);
            l[j] += __shfl_xor_sync(FULL, l[j], 8);
            l[j] += __shfl_xor_sync(FULL, l[j], 16);
            if (lane == 0) s_ml[0][j][warp] = m[j], s_ml[1][j][warp] = l[j];
        }
        __syncthreads();
        // thread (row, dim): their sum, in the warps' order
        const int r = tid / D, dd = tid % D;
        float mx = -INFINITY, ll = 0.0f, x = 0.0f;
        if (r < KO_ROWS) {
#pragma unroll
            for (int i = 0; i < KO_WARPS; i++) mx = fmaxf(mx, s_ml[0][r][i]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int i = 0; i < KO_WARPS; i++) {
                const float f = ex2(s_ml[0][r][i] - ref);
                ll = fmaf(s_ml[1][r][i], f, ll);
                x = fmaf(joined[(i * KO_ROWS + r) * D + dd], f, x);
            }
        }
        auto put = [&](float y, float sum) {
            if (r >= rows) return;
            T* op = static_cast<T*>(a.out) + cc.b * a.o_slot + (r / G) * a.o_row + (cc.h * G + r % G) * a.o_head + dd;
            *op = (T)(sum == 0.0f ? 0.0f : y / sum);
        };
        if (seg_end - seg == cc.tiles) {
            if (r < KO_ROWS) put(x, ll);
        } else {
            constexpr int PART = KO_ROWS * (D + 2);  // [row][dim], then [row][m, l]
            uint32_t* tickets = static_cast<uint32_t*>(a.work);
            float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + KV_TICKETS);
            const int c0 = cut.owner(cc.first), c1 = cut.owner(cc.first + cc.tiles - 1);
            auto of = [&](int i) { return parts + (size_t)(2 * i + (i == c0)) * PART; };
            if (r < KO_ROWS) {
                float* mine = of(cta);
                __stcg(&mine[r * D + dd], x);
                if (dd == 0) __stcg(&mine[KO_ROWS * D + 2 * r], mx), __stcg(&mine[KO_ROWS * D + 2 * r + 1], ll);
                __threadfence();
            }
            __syncthreads();
            if (tid == 0) {
                const bool last = atomicAdd(&tickets[c0], 1u) == (uint32_t)(c1 - c0);
                if (last) tickets[c0] = 0;
                __threadfence();
                s_last = last;
            }
            __syncthreads();
            if (s_last && r < KO_ROWS) {
                float top = -INFINITY, sum = 0.0f, y = 0.0f;
#pragma unroll 8
                for (int i = c0; i <= c1; i++) top = fmaxf(top, __ldcg(&of(i)[KO_ROWS * D + 2 * r]));
                if (top == -INFINITY) top = 0.0f;
#pragma unroll 8  // (the loads of several parts in flight)
                for (int i = c0; i <= c1; i++) {
                    const float* q = of(i);
                    const float f = ex2(__ldcg(&q[KO_ROWS * D + 2 * r]) - top);
                    sum = fmaf(__ldcg(&q[KO_ROWS * D + 2 * r + 1]), f, sum);
                    y = fmaf(__ldcg(&q[r * D + dd]), f, y);
                }
                put(y, sum);
            }
        }
        seg = seg_end;
        __syncthreads();  // (the parts and the rows' table are the next pair's)
    }
    cp_wait<0>();
}

template <int TYPE, int D, class T>
static cudaError_t launch_one(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    constexpr int SMEM = KO_WARPS * KA_RING + KO_WARPS * KO_ROWS * D * 4;
    static PerDeviceOnce once;
    once([] { cudaFuncSetAttribute(k_kv_attn_one<TYPE, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    return kv_launch(k_kv_attn_one<TYPE, D, T>, dim3(a.num_sms), KO_THREADS, SMEM, st, pdl, a);
}
template <int TYPE>
static cudaError_t launch_type(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    if (a.c.d == 128) return a.half ? launch_one<TYPE, 128, __half>(st, a, pdl) : launch_one<TYPE, 128, float>(st, a, pdl);
    return a.half ? launch_one<TYPE, 64, __half>(st, a, pdl) : launch_one<TYPE, 64, float>(st, a, pdl);
}
// at most KA_LINE slots
cudaError_t launch_kv_attention_one(cudaStream_t st, const KvAttnArgs& a, bool pdl) {
    return a.c.type == KV_Q8_0 ? launch_type<KV_Q8_0>(st, a, pdl) : launch_type<KV_Q4_0>(st, a, pdl);
}

}  // namespace ocr
