"""The KV cache in fewer bits and the attentions over it (ocr_op_kv_*, ocr_op_attention_window, ocr_op_attention_tree) on
the B200, against a plain restatement (tests/kv_plain.py: numpy f32 for the quantisers, f64 for the attention).

Tolerances, derived before the first run:
- the cache's rows are compared bit for bit: every rounding of the quantisers is defined;
- f32 rows: a score is a sum of d products of at least 22-bit factors accumulated in f32, so it is off by at most about
  (2^-22 + 2^-21) sum|q k| scale; the inputs keep sum|q k| scale below 24, hence 1.7e-5 in the worst case and a tenth of
  that in practice, beside 2^-22 of the exponential. An output is a mean of values with such weights: 1e-5 of the
  largest |value| that the row may see;
- f16 rows: the weights and the output are rounded to f16, 2^-11 each: 2^-10 of the largest |value|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv_plain as P

pytestmark = pytest.mark.gpu

TYPES = ("f16", "q8_0", "q4_0")
ITEM = {"f32": torch.float32, "f16": torch.float16}
TOL = {"f32": 1e-5, "f16": 2.0 ** -10}


def make_cache(ocr, kind, n_slot, n_kv, n_rows, d, fill=None, **kw):
    """an empty cache of the framework's on the GPU (fill: what its memory holds before)"""
    width, dt = {"f16": (d, torch.float16), "q8_0": (d, torch.int8), "q4_0": (d // 2, torch.uint8)}[kind]
    t = [torch.zeros(n_slot, n_kv, n_rows, width, dtype=dt, device="cuda") for _ in "kv"]
    s = [None, None] if kind == "f16" else \
        [torch.zeros(n_slot, n_kv, n_rows, d // 32, dtype=torch.float16, device="cuda") for _ in "kv"]
    if fill is not None:
        for x in (t if kind == "f16" else s):
            x.fill_(fill)
    torch.cuda.synchronize()
    return ocr.KvCache(kind, t[0], t[1], s[0], s[1], d_head=d, **kw)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sequences(seed, n_slot, n, n_kv, d, item="f32"):
    """keys and values of positions 0 … n - 1 of every slot, [n_slot][n][n_kv][d], on the host"""
    g = np.random.default_rng(seed)
    k = g.standard_normal((n_slot, n, n_kv, d), dtype=np.float32)
    v = g.standard_normal((n_slot, n, n_kv, d), dtype=np.float32) * g.uniform(0.2, 2, (n_slot, n, n_kv, 1)).astype(np.float32)
    if item == "f16":
        k, v = (x.astype(np.float16).astype(np.float32) for x in (k, v))
    return k, v


def put(ocr, ctx, cache, k, v, pos, item="f32", n=None, chunk=None):
    """positions pos[b] … of the sequences → the cache, a call for `chunk` rows"""
    T = k.shape[1]
    chunk = chunk or T
    kd, vd = (torch.from_numpy(x).to("cuda", ITEM[item]) for x in (k, v))
    torch.cuda.synchronize()
    for a in range(0, T, chunk):
        m = min(chunk, T - a)
        left = None if n is None else i32([min(max(x - a, 0), m) for x in n])
        ps = i32([p if p < 0 else p + a for p in pos])
        torch.cuda.synchronize()
        ocr.op_kv_write(ctx, cache, kd[:, a:a + m], vd[:, a:a + m], ps, left)
        ctx.sync()


def awkward(d):
    """rows of blocks that go wrong: zeros, one value, equal magnitudes of both signs, halves, tiny, huge, not finite"""
    g = np.random.default_rng(1)
    rows = [np.zeros(d), np.eye(1, d, d // 3)[0], np.where(np.arange(d) % 2, 1.0, -1.0), np.where(np.arange(d) % 2, -3.0, 3.0),
            np.arange(d) - d / 2 + 0.5, g.standard_normal(d) * 1e-38, g.standard_normal(d) * 6e-8 * 100,
            g.standard_normal(d) * 1e-6, g.standard_normal(d) * 1e4, g.standard_normal(d) * 4e6, g.standard_normal(d) * 1e30]
    for bad in (np.nan, np.inf, -np.inf):
        r = g.standard_normal(d)
        r[d // 2 + 3] = bad
        rows.append(r)
    return np.stack(rows).astype(np.float32)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("kind", TYPES)
def test_rows_are_quantised_as_defined_and_read_back(ocr, ctx, kind, item, d):
    n_slot, n_kv, T, n_rows = 3, 3, 37, 61
    k, v = sequences(5, n_slot, T, n_kv, d)
    k[0, :14, 1], v[1, :14, 0] = awkward(d), awkward(d)
    with np.errstate(over="ignore"):
        if item == "f16":
            k, v = (x.astype(np.float16).astype(np.float32) for x in (k, v))
    cache = make_cache(ocr, kind, n_slot, n_kv, n_rows, d)
    pos, n = [24, -1, 7], [37, 37, 9]
    # strided rows: keys and values side by side, a head apart
    both = torch.zeros(n_slot, T, 2 * n_kv, 2 * d, dtype=ITEM[item], device="cuda")
    both[:, :, 0::2, :d], both[:, :, 1::2, :d] = (torch.from_numpy(x).to("cuda", ITEM[item]) for x in (k, v))
    back = torch.full((n_slot, T, 2 * n_kv, d), 7.0, dtype=ITEM[item], device="cuda")
    ps, ns = i32(pos), i32(n)
    torch.cuda.synchronize()
    ocr.op_kv_write(ctx, cache, both[:, :, 0::2, :d], both[:, :, 1::2, :d], ps, ns)
    ocr.op_kv_read(ctx, cache, back[:, :, :n_kv], back[:, :, n_kv:], ps, ns)
    ctx.sync()
    back = back.float().cpu().numpy()
    for x, got, name in ((k, back[:, :, :n_kv], 0), (v, back[:, :, n_kv:], 1)):
        want = P.held(x, kind)
        for b in range(n_slot):
            m = n[b] if pos[b] >= 0 else 0
            w = want[b, :m]
            if item == "f16":
                with np.errstate(over="ignore"):
                    w = w.astype(np.float16).astype(np.float32)
            np.testing.assert_array_equal(got[b, :m], w)
            assert (got[b, m:] == 0).all()
        # the bytes themselves, and that nothing else was touched
        raw = cache._keep[name].cpu().numpy()
        if kind == "f16":
            with np.errstate(over="ignore"):
                rows = x.astype(np.float16)
            scales = None
        else:
            q, scales = P.quantise(x, kind)
            rows = P.packed(q, kind)
            raw_s = cache._keep[2 + name].cpu().numpy()
        for b in range(n_slot):
            m, p = (n[b], pos[b]) if pos[b] >= 0 else (0, 0)
            np.testing.assert_array_equal(raw[b, :, p:p + m], rows[b, :m].transpose(1, 0, 2))
            assert not raw[b, :, :p].any() and not raw[b, :, p + m:].any()
            if scales is not None:
                np.testing.assert_array_equal(raw_s[b, :, p:p + m], scales[b, :m].transpose(1, 0, 2))


# slots, kv heads, query heads per kv head, d, rows, positions before them, window, sinks, ring, a tree
SHAPES = [
    (1, 1, 1, 128, 1, [0], 0, 0, False, False),            # the first token
    (1, 2, 2, 128, 1, [1], 0, 0, False, False),
    (2, 1, 8, 64, 1, [63, 200], 0, 0, False, False),
    (3, 2, 3, 128, 1, [300, -1, 17], 0, 0, False, False),  # an idle slot, groups of three
    (4, 2, 2, 128, 1, [515, 31, 64, 129], 100, 5, False, False),
    (2, 2, 1, 64, 1, [700, 90], 1, 0, False, False),       # a row sees itself alone
    (2, 1, 2, 128, 1, [900, 37], 64, 4, True, False),
    (1, 1, 16, 64, 3, [77], 33, 40, False, False),
    (2, 2, 2, 64, 5, [250, 0], 0, 0, False, False),
    (2, 1, 4, 128, 7, [431, 12], 50, 3, True, False),
    (1, 2, 2, 128, 33, [100], 0, 0, False, False),
    (2, 1, 2, 64, 100, [0, 77], 0, 0, False, False),       # a prompt from its start
    (1, 1, 3, 128, 150, [41], 64, 2, False, False),
    (1, 2, 8, 64, 67, [260], 90, 16, True, False),
    (1, 1, 1, 128, 300, [0], 10, 0, False, False),
    (1, 1, 2, 128, 2, [300], 0, 0, False, True),
    (3, 2, 2, 128, 8, [200, 3, -1], 0, 0, False, True),
    (2, 1, 4, 64, 16, [513, 0], 0, 0, False, True),        # a tree before anything is committed
    (1, 2, 2, 64, 29, [140], 20, 2, False, True),
    (2, 1, 3, 128, 64, [90, 259], 0, 0, False, True),
    (1, 1, 8, 128, 61, [333], 40, 7, True, True),
]


def tree(seed, T):
    g = np.random.default_rng(seed)
    return [-1] + [int(g.integers(max(-1, i - 1 - int(g.choice([0, 1, 4, 16]))), i)) for i in range(1, T)]


def case(ocr, ctx, kind, item, shape, seed=3, n=None, fill=None, spare=5, change=None, q_scale=1.0):
    """→ (out, want, largest |value|, cache) of one call"""
    n_slot, n_kv, G, d, T, pos, window, sinks, ring, drafts = shape
    total = max(pos) + T
    k, v = sequences(seed, n_slot, total, n_kv, d, item)
    q = np.random.default_rng(seed + 1).standard_normal((n_slot, T, n_kv * G, d), dtype=np.float32) * q_scale
    if change is not None:
        change(k, v)
    n_rows = sinks + window + max(T, 16) - 1 + spare if ring else total + spare
    cache = make_cache(ocr, kind, n_slot, n_kv, n_rows, d, fill=fill, window=window, sinks=sinks, ring=ring)
    put(ocr, ctx, cache, k, v, [0 if p >= 0 else -1 for p in pos], item, [p + T for p in pos], 16 if ring else None)
    parents = [tree(seed + b, T) for b in range(n_slot)] if drafts else [None] * n_slot
    qkv = torch.zeros(n_slot, T, n_kv * G + 2, d, dtype=ITEM[item], device="cuda")  # rows with a gap between them
    qkv[:, :, :n_kv * G] = torch.from_numpy(q)
    out = torch.full((n_slot, n_kv * G, T, d), 7.0, dtype=ITEM[item], device="cuda").transpose(1, 2)
    ps, ns, scale = i32(pos), None if n is None else i32(n), 1.0 / math.sqrt(d)
    par = i32(parents) if drafts else None
    torch.cuda.synchronize()

    def call():
        if drafts:
            ocr.op_attention_tree(ctx, cache, qkv[:, :, :n_kv * G], out, ps, par, scale, ns)
        else:
            ocr.op_attention_window(ctx, cache, qkv[:, :, :n_kv * G], out, ps, scale, ns)
        ctx.sync()
        return out.double().cpu()

    want = torch.zeros(n_slot, T, n_kv * G, d, dtype=torch.float64)
    qd = qkv[:, :, :n_kv * G].double().cpu()
    top = 0.0
    for b in range(n_slot):
        m = T if n is None else n[b]
        if pos[b] < 0 or m == 0:
            continue
        kb, vb = (torch.from_numpy(P.held(x[b, :pos[b] + m], kind)).double().transpose(0, 1) for x in (k, v))
        top = max(top, float(vb.abs().nan_to_num(0, 0, 0).max()))
        want[b, :m] = P.attend(qd[b, :m], kb, vb, pos[b], scale, window, sinks,
                               None if parents[b] is None else parents[b][:m])
    return call, want, top


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)).replace(" ", ""))
@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("kind", TYPES)
def test_attention_matches_the_formula(ocr, ctx, kind, item, shape):
    call, want, top = case(ocr, ctx, kind, item, shape)
    got = call()
    err = float((got - want).abs().max()) / top
    assert err <= TOL[item], f"{err:.2e} of the largest value"
    assert torch.equal(got, call())  # the same bits again


# many tiles to a CTA, triples cut in pieces and taken whole, more (slot, row block) pairs than the line holds, more slots
LONG = [
    (3, 8, 2, 128, 1, [5000, 3000, 4100], 0, 0, False, False),
    (2, 8, 4, 64, 1, [9000, 8700], 6000, 64, True, False),
    (600, 1, 2, 64, 1, list(range(600)), 0, 0, False, False),
    (1, 8, 2, 128, 16, [2303], 0, 0, False, True),
    (2, 8, 2, 128, 8, [3000, 2900], 0, 0, False, True),
    (2, 8, 4, 128, 61, [3000, 2000], 1024, 16, False, True),
    (1, 8, 2, 128, 700, [1500], 0, 0, False, False),
    (2, 4, 4, 64, 300, [3100, 2500], 0, 0, False, False),
    (1, 8, 2, 128, 1500, [0], 300, 5, False, False),
    (1, 4, 2, 64, 500, [2000], 700, 9, True, False),
    (40, 1, 1, 64, 1700, [0, 7] * 20, 0, 0, False, False),
]


@pytest.mark.parametrize("shape", LONG, ids=lambda s: "-".join(map(str, s)).replace(" ", "")[:60])
@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("kind", TYPES)
def test_long_attention_matches_the_formula(ocr, ctx, kind, item, shape):
    if shape[0] > 8 and (kind, item) not in (("f16", "f32"), ("q4_0", "f16")):
        pytest.skip("the schedule is the same for every type")
    call, want, top = case(ocr, ctx, kind, item, shape)
    got = call()
    err = float((got - want).abs().max()) / top
    assert err <= TOL[item], f"{err:.2e} of the largest value"
    assert torch.equal(got, call())


# a slot's rows past one launch's share of (slot, row block) pairs
def test_more_slots_than_a_launch_takes(ocr, ctx):
    shape = (4100, 1, 1, 64, 33, [i % 50 for i in range(4100)], 0, 0, False, False)
    call, want, top = case(ocr, ctx, "f16", "f16", shape)
    assert float((call() - want).abs().max()) / top <= TOL["f16"]


# many tiles to a whole (row block, kv head), the scores rising (so the reference moves between tiles) or falling
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_along_a_long_cache(ocr, ctx, kind, rising):
    shape = (1, 8, 2, 128, 700, [3000], 0, 0, False, False)

    def change(k, v):
        f = np.linspace(0.05, 3.0, k.shape[1], dtype=np.float32)
        k *= (f if rising else f[::-1])[None, :, None, None]

    call, want, top = case(ocr, ctx, kind, "f32", shape, change=change)
    got = call()
    assert float((got - want).abs().max()) / top <= TOL["f32"]
    assert torch.equal(got, call())


def test_the_plain_mask_is_its_definition():
    for pos, T, window, sinks, parent in ((7, 5, 0, 0, None), (20, 6, 8, 3, None), (3, 9, 4, 5, tree(1, 9)), (30, 12, 10, 2, tree(2, 12))):
        m = P.mask_of(pos, T, window, sinks, parent)
        assert m.tolist() == [[P.sees(pos, t, j, window, sinks, parent) for j in range(pos + T)] for t in range(T)]


@pytest.mark.parametrize("kind", TYPES)
def test_rows_not_in_use_are_zeros(ocr, ctx, kind):
    for shape, n in (((3, 2, 2, 128, 6, [100, 40, -1], 0, 0, False, False), [4, 0, 6]),
                     ((2, 1, 2, 64, 150, [30, 200], 64, 4, False, False), [130, 1]),
                     ((2, 1, 4, 64, 40, [50, 7], 0, 0, False, True), [0, 33])):
        call, want, top = case(ocr, ctx, kind, "f32", shape, n=n)
        got = call()
        assert float((got - want).abs().max()) / top <= TOL["f32"]
        for b, m in enumerate(n):
            assert (got[b, m if shape[5][b] >= 0 else 0:] == 0).all()


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (3, 4, 6, 7, 8, 9, 12, 13, 18, 19, 20)],
                         ids=lambda s: "-".join(map(str, s)).replace(" ", ""))
@pytest.mark.parametrize("kind", TYPES)
def test_what_a_row_does_not_see_has_no_part(ocr, ctx, kind, shape):
    """memory that no row was written to holds NaN (in the scales of the quantised types, in the rows of f16); positions
    outside some rows' view hold infinities and NaN: rows that do not see them are right, rows that do are not finite"""
    n_slot, n_kv, G, d, T, pos, window, sinks, ring, drafts = shape
    live = [b for b in range(n_slot) if pos[b] >= 0]
    hit = {}

    def change(k, v):
        for b in live:  # one position that the last row sees, if it is not the first row too: the one before last
            j = pos[b] + T // 2
            hit[b] = j
            k[b, j, 0, 3], v[b, j, n_kv - 1, 5] = np.nan, np.inf if b % 2 else np.nan

    call, want, top = case(ocr, ctx, kind, "f32", shape, fill=float("nan"), change=change)
    got = call()
    parents = [tree(3 + b, T) for b in range(n_slot)] if drafts else [None] * n_slot
    for b in live:
        for t in range(T):
            seen = P.sees(pos[b], t, hit[b], window, sinks, parents[b])
            for h in range(n_kv * G):
                touched = seen and (h // G == 0 or h // G == n_kv - 1)
                if touched:
                    assert not torch.isfinite(got[b, t, h]).all()
                else:
                    assert float((got[b, t, h] - want[b, t, h]).abs().max()) / top <= TOL["f32"], (b, t, h)


@pytest.mark.parametrize("T", [1, 130])
@pytest.mark.parametrize("kind", TYPES)
def test_large_and_small_magnitudes(ocr, ctx, kind, T):
    """values and keys whose size changes from position to position by many powers of two, queries of any size"""
    def change(k, v):
        e = np.random.default_rng(9).integers(-12, 10, v.shape[:3] + (1,)).astype(np.float32)
        v *= np.exp2(e)
        k *= np.exp2(np.float32(-9))

    call, want, top = case(ocr, ctx, kind, "f32", (2, 1, 2, 128, T, [300, 77], 0, 0, False, False), change=change,
                           q_scale=512.0)
    assert float((call() - want).abs().max()) / top <= TOL["f32"]

    def small(k, v):
        v *= np.float32(2.0 ** -9)

    call, want, top = case(ocr, ctx, kind, "f32", (1, 1, 2, 128, T, [300], 0, 0, False, False), change=small,
                           q_scale=2.0 ** -14)
    assert float((call() - want).abs().max()) / top <= TOL["f32"]


@pytest.mark.parametrize("kind", ["f16", "q4_0"])
def test_scores_far_apart(ocr, ctx, kind):
    """one key far above the others, late: every weight before it vanishes; far below: nothing overflows"""
    for up in (40.0, -40.0):
        def change(k, v):
            k[:, -20] *= up

        call, want, top = case(ocr, ctx, kind, "f32", (1, 1, 2, 64, 129, [400], 0, 0, False, False), change=change)
        # (scores of 40 x the others': the products' sum grows alike, and so does the bound)
        assert float((call() - want).abs().max()) / top <= 40 * TOL["f32"]


def test_offsets_past_32_bits(ocr, ctx):
    """a cache of 2.1 billion elements and 4.3 GB per tensor: the last head's last rows"""
    n_kv, n_rows, d = 9, 1 << 21, 128
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("not enough memory")
    cache = make_cache(ocr, "f16", 1, n_kv, n_rows, d, window=200, sinks=3)
    pos = n_rows - 310
    k, v = sequences(2, 1, 310, n_kv, d)
    put(ocr, ctx, cache, k, v, [pos])
    ks, vs = sequences(4, 1, 3, n_kv, d)
    put(ocr, ctx, cache, ks, vs, [0])
    for T in (1, 8, 100):
        q = torch.randn(1, T, 2 * n_kv, d, device="cuda")
        out = torch.empty_like(q)
        ps = i32([n_rows - T])
        torch.cuda.synchronize()
        ocr.op_attention_window(ctx, cache, q, out, ps, 0.1)
        ctx.sync()
        # the same rows as a short sequence: the sinks, then the last 310 positions
        kk, vv = (torch.from_numpy(np.concatenate([P.held(a[0], "f16"), P.held(b[0], "f16")])).double().transpose(0, 1)
                  for a, b in ((ks, k), (vs, v)))
        want = P.attend(q[0].double().cpu(), kk, vv, 313 - T, 0.1, 200, 3)
        assert float((out[0].double().cpu() - want).abs().max() / vv.abs().max()) <= TOL["f32"]


@pytest.mark.parametrize("kind", TYPES)
def test_accepted_rows_move_together(ocr, ctx, kind):
    n_slot, n_kv, d, T = 3, 2, 128, 12
    paths = [[0, 2, 3, 9, 11], [5], list(range(12))]
    pos = [30, 7, -1]
    for ring in (False, True):
        n_rows, kw = (60, {}) if not ring else (33, dict(window=16, sinks=4, ring=True))
        caches = [make_cache(ocr, kind, n_slot, n_kv, n_rows, d, **kw) for _ in range(3)]
        seqs = [sequences(20 + i, n_slot, T, n_kv, d) for i in range(3)]
        for c, (k, v) in zip(caches, seqs):
            put(ocr, ctx, c, k, v, [p if p >= 0 else 0 for p in pos])
        before = [[t.clone() for t in c._keep if t is not None] for c in caches]
        path = i32([p + [0] * (T - len(p)) for p in paths])
        n, ps = i32([len(p) for p in paths]), i32(pos)
        torch.cuda.synchronize()
        ocr.op_kv_keep(ctx, caches, ps, path, n)
        ctx.sync()
        for c, old in zip(caches, before):
            for now, was in zip([t for t in c._keep if t is not None], old):
                want = was.clone()
                for b in range(n_slot):
                    if pos[b] < 0:
                        continue
                    for i, j in enumerate(paths[b]):
                        want[b, :, P.row_of(pos[b] + i, n_rows, kw.get("sinks", 0), ring)] = \
                            was[b, :, P.row_of(pos[b] + j, n_rows, kw.get("sinks", 0), ring)]
                assert torch.equal(now, want)


def test_a_captured_step_replays_as_the_sequences_grow(ocr, ctx):
    """write + attention in a CUDA graph: positions are device memory, so one capture serves every step"""
    n_kv, d, n = 2, 128, 40
    k, v = sequences(8, 2, n, n_kv, d)
    cache, want_cache = (make_cache(ocr, "q8_0", 2, n_kv, 64, d, window=16, sinks=2) for _ in range(2))
    kd, vd = (torch.zeros(2, 1, n_kv, d, device="cuda") for _ in "kv")
    q, out, ps = torch.randn(2, 1, 4, d, device="cuda"), torch.zeros(2, 1, 4, d, device="cuda"), i32([0, 0])
    stream = torch.cuda.ExternalStream(ctx.stream())

    def step(c):
        ocr.op_kv_write(ctx, c, kd, vd, ps)
        ocr.op_attention_window(ctx, c, q, out, ps, 0.09)

    torch.cuda.synchronize()
    step(want_cache)  # (the workspace is made before the capture)
    ctx.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step(cache)
    for i in range(n):
        kd.copy_(torch.from_numpy(k[:, i:i + 1]))
        vd.copy_(torch.from_numpy(v[:, i:i + 1]))
        ps.fill_(i)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        ctx.sync()
        got = out.clone()
        step(want_cache)
        ctx.sync()
        assert torch.equal(got, out)
    kk, vv = (torch.from_numpy(P.held(x[1], "q8_0")).double().transpose(0, 1) for x in (k, v))
    want = P.attend(q[1].double().cpu(), kk, vv, n - 1, 0.09, 16, 2)
    assert float((got[1].double().cpu() - want).abs().max() / vv.abs().max()) <= TOL["f32"]
    del g


def test_rows_made_on_another_stream(ocr, ctx):
    """the context's stream waits for the caller's by an event, as the interface says"""
    n_kv, d, T = 2, 64, 50
    cache = make_cache(ocr, "q4_0", 1, n_kv, 200, d)
    k, v = sequences(6, 1, T, n_kv, d)
    mine, theirs = torch.cuda.Stream(), torch.cuda.ExternalStream(ctx.stream())
    kd, vd, back = (torch.zeros(1, T, n_kv, d, device="cuda") for _ in range(3))
    bv, ps = torch.zeros_like(back), i32([3])
    hk, hv = (torch.from_numpy(x).pin_memory() for x in (k, v))
    torch.cuda.synchronize()
    with torch.cuda.stream(mine):
        torch.cuda._sleep(20_000_000)
        kd.copy_(hk, non_blocking=True)
        vd.copy_(hv, non_blocking=True)
    theirs.wait_stream(mine)
    ocr.op_kv_write(ctx, cache, kd, vd, ps)
    ocr.op_kv_read(ctx, cache, back, bv, ps)
    mine.wait_stream(theirs)
    with torch.cuda.stream(mine):
        got = back.clone()
    torch.cuda.synchronize()
    np.testing.assert_array_equal(got.cpu().numpy(), P.held(k, "q4_0"))


def test_a_sessions_layer_as_a_cache(ocr, ctx):
    """a live session's f16 rows read through the view, quantised into a q8_0 cache, and attended from both"""
    cfg = ocr.TextConfig(n_layer=2, dim=256, n_head=2, n_kv=1, d_head=128, n_ff=512, n_vocab=1000, n_ctx_train=4096)
    m = ocr.TextModel.synthetic(ctx, cfg, 7, 0.2, 1.0)
    s = m.session(64, 2)
    s.prefill(1, ids=[int(x) for x in ocr.fill_ids(3, 40, 1000)])
    live = s.kv_cache(1)
    assert (live.c.n_slot, live.c.n_kv, live.c.n_rows, live.c.d_head) == (2, 1, 64, 128)
    k, v = (torch.zeros(2, 40, 1, 128, device="cuda") for _ in "kv")
    ps = i32([-1, 0])
    torch.cuda.synchronize()
    ocr.op_kv_read(ctx, live, k, v, ps)
    ctx.sync()
    hk, hv = s.kv(1, 1, 0, 40)
    np.testing.assert_array_equal(k[1, :, 0].cpu().numpy(), hk.view(np.float16).astype(np.float32))
    np.testing.assert_array_equal(v[1, :, 0].cpu().numpy(), hv.view(np.float16).astype(np.float32))
    q8 = make_cache(ocr, "q8_0", 2, 1, 64, 128)
    ocr.op_kv_write(ctx, q8, k, v, ps)
    q, out, at = torch.randn(2, 1, 2, 128, device="cuda"), torch.zeros(2, 1, 2, 128, device="cuda"), i32([-1, 39])
    torch.cuda.synchronize()
    for cache, kind in ((live, "f16"), (q8, "q8_0")):
        ocr.op_attention_window(ctx, cache, q, out, at, 0.088)
        ctx.sync()
        kk, vv = (torch.from_numpy(P.held(x[1].cpu().numpy(), kind)).double().transpose(0, 1) for x in (k, v))
        want = P.attend(q[1].double().cpu(), kk, vv, 39, 0.088)
        # (the synthetic model's keys are larger than the other tests': the scores' sums of products reach 100)
        assert float((out[1].double().cpu() - want).abs().max() / vv.abs().max()) <= 5 * TOL["f32"]
    s.close()
    m.close()


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_arguments_are_refused(ocr, ctx):
    def rows(T=2, n_kv=2, d=128, n_slot=2, dt=torch.float32):
        return torch.zeros(n_slot, T, n_kv, d, dtype=dt, device="cuda")

    cache = make_cache(ocr, "q8_0", 2, 2, 32, 128)
    ps = i32([0, 0])
    k = rows()

    def refused(match, f, *a, **kw):
        with pytest.raises(ocr.OcrError, match=match):
            f(*a, **kw)

    refused("cache type", ocr.KvCache, "q5_0", k, k)
    refused("contiguous", ocr.KvCache, "f16", k.half(), k.half(), d_head=64)
    refused("contiguous", ocr.KvCache, "q8_0", cache._keep[0], cache._keep[1])  # no scales
    refused("rows must be", ocr.op_kv_write, ctx, cache, rows(d=64), rows(d=64), ps)
    refused("rows must be", ocr.op_kv_write, ctx, cache, rows(n_kv=3), rows(n_kv=3), ps)
    refused("rows must be", ocr.op_kv_write, ctx, cache, rows(dt=torch.bfloat16), rows(dt=torch.bfloat16), ps)
    refused("one type", ocr.op_kv_write, ctx, cache, k, k.half(), ps)
    refused("one shape", ocr.op_kv_write, ctx, cache, k, rows(T=3), ps)
    refused("int32", ocr.op_kv_write, ctx, cache, k, k, ps.long())
    refused("int32", ocr.op_kv_write, ctx, cache, k, k, i32([0]))
    refused("more than the cache", ocr.op_kv_write, ctx, cache, rows(T=33), rows(T=33), ps)
    off = torch.zeros(2 * 2 * 2 * 128 + 4, device="cuda")
    refused("16 bytes", ocr.op_kv_write, ctx, cache, off[1:1025].view(2, 2, 2, 128), k, ps)
    refused("16 bytes", ocr.op_kv_read, ctx, cache, k, torch.zeros(2, 2, 2, 130, device="cuda")[..., :128], ps)
    q = rows(n_kv=4)
    refused("multiple of n_kv", ocr.op_attention_window, ctx, cache, rows(n_kv=3), rows(n_kv=3), ps, 0.1)
    refused("scale", ocr.op_attention_window, ctx, cache, q, q, ps, float("nan"))
    refused("scale", ocr.op_attention_window, ctx, cache, q, q, ps, 0.0)
    refused("one type", ocr.op_attention_window, ctx, cache, q, q.half(), ps, 0.1)
    long = make_cache(ocr, "q8_0", 2, 2, 100, 128)
    q65 = rows(T=65, n_kv=4)
    refused("at most 64", ocr.op_attention_tree, ctx, long, q65, q65, ps, torch.zeros(2, 65, dtype=torch.int32,
                                                                                    device="cuda"), 0.1)
    refused("at most 64", ocr.op_kv_keep, ctx, [long], ps, torch.zeros(2, 65, dtype=torch.int32, device="cuda"), ps)
    refused("one shape", ocr.op_kv_keep, ctx, [long, cache], ps, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ps)
    wide = torch.zeros(1, 65537, 8, 64, dtype=torch.float16, device="cuda")
    refused("more than one launch", ocr.op_attention_window, ctx, make_cache(ocr, "q4_0", 1, 1, 65537, 64), wide, wide,
            i32([0]), 0.1)
    ring = make_cache(ocr, "q8_0", 2, 2, 32, 128, window=20, sinks=4, ring=True)
    refused("more than the cache", ocr.op_kv_write, ctx, ring, rows(T=10), rows(T=10), ps)
    refused("ring cache", ocr.op_kv_write, ctx, make_cache(ocr, "q8_0", 2, 2, 32, 128, ring=True), k, k, ps)
    refused("ring cache", ocr.op_kv_write, ctx, make_cache(ocr, "q8_0", 2, 2, 32, 128, window=30, sinks=4, ring=True), k,
            k, ps)
    refused("64 or 128", ocr.op_kv_write, ctx,
            ocr.KvCache("f16", *(torch.zeros(2, 2, 8, 96, dtype=torch.float16, device="cuda") for _ in "kv"), d_head=96),
            rows(d=96), rows(d=96), ps)
    ctx.sync()  # nothing was launched, nothing is flagged


@pytest.mark.parametrize("T", [2, 70])
def test_positions_outside_the_cache_are_flagged(ocr, ctx, T):
    """the slot concerned is left alone, the others are served, the next sync says so, the one after is clean"""
    cache = make_cache(ocr, "q8_0", 2, 1, 100, 128)
    k, v = sequences(1, 2, T, 1, 128)
    kd, vd = (torch.from_numpy(x).cuda() for x in (k, v))
    ps = i32([100 - T + 1, 5])
    torch.cuda.synchronize()
    ocr.op_kv_write(ctx, cache, kd, vd, ps)
    with pytest.raises(ocr.OcrError, match="position outside"):
        ctx.sync()
    assert not cache._keep[0][0].any() and cache._keep[0][1, :, 5:5 + T].any()
    q = torch.randn(2, T, 2, 128, device="cuda")
    out = torch.full_like(q, 7.0)
    torch.cuda.synchronize()
    ocr.op_attention_window(ctx, cache, q, out, ps, 0.1)
    with pytest.raises(ocr.OcrError, match="position outside"):
        ctx.sync()
    assert not out[0].any() and out[1].any() and torch.isfinite(out[1]).all()
    ctx.sync()


@pytest.mark.parametrize("T", [6, 40])
def test_trees_and_paths_that_are_none_are_flagged(ocr, ctx, T):
    cache = make_cache(ocr, "f16", 2, 1, 100, 64)
    q = torch.randn(2, T, 2, 64, device="cuda")
    out = torch.empty_like(q)
    good = list(range(-1, T - 1))
    ps = i32([5, 5])
    for bad in ([good[0], 1] + good[2:], [good[0], T] + good[2:], [-2] + good[1:]):
        par = i32([bad, good])
        torch.cuda.synchronize()
        ocr.op_attention_tree(ctx, cache, q, out, ps, par, 0.1)
        with pytest.raises(ocr.OcrError, match="index outside"):
            ctx.sync()
    for path, n in (([0, 2, 2], 3), ([3, 1, 4], 3), ([0, 1, T], 3), ([-1, 1, 2], 3)):
        before = cache._keep[0].clone()
        p = i32([path + [0] * (T - 3), [0] * T])
        ns = i32([n, 0])
        torch.cuda.synchronize()
        ocr.op_kv_keep(ctx, [cache], ps, p, ns)
        with pytest.raises(ocr.OcrError, match="index outside"):
            ctx.sync()
        assert torch.equal(before, cache._keep[0])
    ns = i32([T + 1, 0])
    p = i32([good, good])
    torch.cuda.synchronize()
    ocr.op_kv_keep(ctx, [cache], ps, p, ns)
    with pytest.raises(ocr.OcrError, match="position outside"):
        ctx.sync()
    ctx.sync()
