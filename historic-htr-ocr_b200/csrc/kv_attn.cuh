// kv_attn.cuh — what the three attentions over a KV cache share (k_kv_attn_one.cu, k_kv_attn.cu: a few rows per kv head;
// k_kv_attn_tc.cu: many): the line of key tiles that is cut evenly over the CTAs, the positions that a range of rows sees,
// the quants' way to f16.
#pragma once

#include "kv.cuh"

namespace ocr {

constexpr int KV_LINE = 4096;     // (slot, row block) pairs whose prefix sums a CTA holds (k_kv_attn_tc.cu)
constexpr int KA_LINE = 256;      // slots of a launch of the attentions of few rows
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// the remainders of a and b past their f16 rounding `hi`
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t hi) {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack2(a - h.x, b - h.y);
}
// A query's values a and b in f16 hi (→) + lo (rest2) whose products with an infinite key are infinities of one sign, as the
// value's own: hi is rounded towards zero from a little less than the value, so lo is of its sign and not zero either
// (values above 2^-24 of the row's largest, which is scaled to 2^10 … 2^11).
__device__ __forceinline__ uint32_t pack2_below(float a, float b) {
    uint32_t hi;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(__fmul_rz(b, 0.99999994f)), "f"(__fmul_rz(a, 0.99999994f)));
    return hi;
}
// an unsigned byte pair placed as halves of 1024 + u, less `bias`
__device__ __forceinline__ uint32_t bytes_h2(uint32_t w, uint32_t sel, uint32_t bias) {
    const uint32_t m = __byte_perm(w, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t H2_1152 = 0x64806480u;  // 1024 + 128: an int8 with its sign bit flipped
// the low (SHIFT = 0) or high nibbles of bytes 0 and 2 of w, less 8
template <bool HIGH>
__device__ __forceinline__ uint32_t nibbles_h2(uint32_t w) {
    const uint32_t m = (w & (HIGH ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;  // 1024 + n, or 1024 + 16 n
    const __half2 x = *reinterpret_cast<const __half2*>(&m);
    __half2 r;
    if (HIGH)
        r = __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-72.0f));
    else
        r = __hsub2(x, __float2half2_rn(1032.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// the keys that rows t0 … t1 - 1 of a slot's call see together, in order: the sinks that lie before the first row's
// window, then positions lo … end - 1 (drafts: every row may stand at the first position)
struct KvSpan {
    int pos, m, lo, ns, nv;  // m: the slot's rows in use
    __device__ __forceinline__ void set(const KvAttnArgs& a, int b, int t0, int t1) {
        set(a, a.r.pos[b], a.r.rows(a.c, b, a.err), t0, t1);
    }
    __device__ __forceinline__ void set(const KvAttnArgs& a, int pos_, int m_, int t0, int t1) {
        pos = pos_, m = m_;
        const int first = pos + (a.parent ? 0 : t0);
        lo = a.c.window ? max(0, first - a.c.window + 1) : 0;
        ns = min(a.c.sinks, lo);
        nv = t0 < m ? ns + pos + (a.parent ? m : min(t1, m)) - lo : 0;
    }
    __device__ __forceinline__ int position(int v) const { return v < ns ? v : lo + v - ns; }
};

// which keys of a span a row sees, as up to two ranges and, for drafts, a set
struct KvSight {
    int a, lo, hi;  // keys 0 … a - 1 and lo … hi - 1 of the span
    int draft;      // the key of the first draft
    uint64_t set;   // the drafts that the row sees
    // a row at position `at`, which sees positions up to `last`
    __device__ __forceinline__ void rows(const KvView& c, const KvSpan& s, int at, int last) {
        const int shift = s.ns - s.lo;  // key = position + shift, from the window on
        hi = min(s.nv, last + 1 + shift);
        lo = c.window ? max(0, at - c.window + 1 + shift) : 0;
        a = min(hi, max(s.ns, c.sinks + shift));
        draft = s.pos + shift;
        set = 0;
    }
    // of keys v … v + 31, those that the row sees
    __device__ __forceinline__ uint32_t mask(int v) const {
        auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
        uint32_t m = below(a - v) | (below(hi - v) & ~below(lo - v));
        const int sh = v - draft;
        if (set && sh > -32 && sh < 64) m |= sh >= 0 ? (uint32_t)(set >> sh) : (uint32_t)(set << -sh);
        return m;
    }
};
// a draft's place: its depth (position pos + depth) and what it sees; parent and depth of the slot's drafts may be read
__device__ __forceinline__ void kv_draft(const KvView& c, const KvSpan& s, int row, const int* parent, const int* depth,
                                         KvSight& sight) {
    const int at = s.pos + depth[row];
    sight.rows(c, s, at, s.pos - 1);
    for (int i = row; i >= 0;) {
        const int where = s.pos + depth[i];
        if (!c.window || where > at - c.window || where < c.sinks) sight.set |= 1ull << i;
        i = parent[i] < i ? parent[i] : -1;
    }
}
__device__ __forceinline__ int kv_depth(int row, const int* parent, int* err) {
    int d = -1;
    for (int i = row; i >= 0; d++) {
        const int p = parent[i];
        if (p >= i || p < -1) dev_error(err, DEV_BAD_INDEX);  // (then taken for a child of the committed rows)
        i = p < i ? p : -1;
    }
    return d;
}

// The least tiles of a part. A pair in p parts takes its tiles' time / p and p parts to join, a part's join about a
// quarter of a tile's time for `at_once` tiles side by side: p near the root of the pair's tiles.
__device__ __forceinline__ int kv_least_share(int total, int pairs, int at_once) {
    return at_once * max(1, (int)(0.75f * sqrtf((float)total / (float)max(pairs, 1) / (float)at_once)));
}
// the line of tiles cut into parts of one size, or one more: CTA i takes tiles part(i) … part(i + 1) - 1
struct KvLine {
    int n, size, more;  // parts, tiles of each, the first `more` of them have another
    __device__ __forceinline__ void cut(int total, int parts) { n = parts, size = total / max(parts, 1), more = total - size * parts; }
    __device__ __forceinline__ int part(int i) const { return i * size + min(i, more); }
    __device__ __forceinline__ int owner(int tile) const {
        const int t = tile - more * (size + 1);
        return t < 0 ? tile / (size + 1) : more + t / size;
    }
};

// The tiles begin … end - 1 of CTA i: an even part of the line, or whole pairs (`per` to an entry of prefix) where those
// take less. Costs in tiles: `piece` for a pair or a piece of one beside its tiles, `join` for the two that are cut.
__device__ __forceinline__ void kv_share(const KvLine& cut, int i, const int* prefix, int entries, int per, int total, int longest,
                                         int grid, int piece, int join, int& begin, int& end) {
    const int pairs = entries * per, each = (pairs + grid - 1) / grid, share = total / grid + 1;
    const long whole_cost = (long)each * (longest + piece);
    const long cut_cost = share + (long)piece * (1 + (long)share * pairs / max(total, 1)) + 2L * join;
    begin = end = 0;
    if (whole_cost <= cut_cost) {
        auto start = [&](int t) {  // the first tile of pair t
            if (t >= pairs) return total;
            const int e = t / per;
            return prefix[e] + t % per * ((prefix[e + 1] - prefix[e]) / per);
        };
        begin = start(i * each), end = start((i + 1) * each);
    } else if (i < cut.n) {
        begin = cut.part(i), end = cut.part(i + 1);
    }
}

// where a CTA stands in the line of tiles
struct KvCursor {
    int b, h, first, tiles;  // the entry and the kv head, the first of its tiles in the line, their number
    __device__ __forceinline__ void at(int g, const int* prefix, int n, int n_kv) {  // the pair of tile g
        int lo = 0, hi = n;  // prefix[lo] <= g < prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= g)
                lo = mid;
            else
                hi = mid;
        }
        b = lo;
        tiles = (prefix[b + 1] - prefix[b]) / n_kv;
        h = (g - prefix[b]) / tiles;
        first = prefix[b] + h * tiles;
    }
};

}  // namespace ocr
