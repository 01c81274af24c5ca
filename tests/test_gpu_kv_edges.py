"""The KV cache operators where they can go wrong apart from their formulas' ordinary cases: captured steps beside other
calls, the context's state after an error, the last rows of a cache, numbers far apart, arguments that are no device
memory. Tolerances are those of test_gpu_kv.py unless a test derives its own."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import kv_plain as P
import test_gpu_kv as common
from test_gpu_kv import ITEM, TOL, TYPES, case, i32, make_cache, put, sequences, tree

pytestmark = pytest.mark.gpu


# ---- the workspace ----
def attend(ocr, ctx, T, n_slot=1, keys=2000, d=128, kind="q8_0", seed=0):
    """a window attention's call over a cache of some contents → (call, out, the tensors it works on)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = make_cache(ocr, kind, n_slot, 2, keys + T, d)
    k, v = (torch.randn(n_slot, keys + T, 2, d, device="cuda", generator=g) for _ in "kv")
    q = torch.randn(n_slot, T, 4, d, device="cuda", generator=g)
    out, zero, ps = torch.zeros_like(q), i32([0] * n_slot), i32([keys] * n_slot)
    torch.cuda.synchronize()
    ocr.op_kv_write(ctx, cache, k, v, zero)
    ctx.sync()
    return lambda: ocr.op_attention_window(ctx, cache, q, out, ps, 0.09), out, (cache, q, ps)


def test_the_workspace_does_not_depend_on_the_call(ocr):
    ctx = ocr.Context(0)
    held = set()
    for T, d in ((1, 64), (16, 128), (130, 64), (300, 128)):
        call, _, keep = attend(ocr, ctx, T, d=d)
        call()
        ctx.sync()
        held.add(ctx.memory()["work"])
    assert len(held) == 1 and held.pop() > 0
    ctx.close()


def test_a_captured_step_replays_after_larger_calls(ocr):
    """a decode step and a tree-sized one captured, then prompts on the same context (pairs cut over many CTAs, so that
    both use the tickets and the partial results), then the replays: the same bits as before"""
    ctx = ocr.Context(0)
    stream = torch.cuda.ExternalStream(ctx.stream())
    steps = [attend(ocr, ctx, T, keys=6000, d=64) for T in (1, 8)]
    larger = [attend(ocr, ctx, T, n_slot=2, keys=1000 + T, d=128) for T in (100, 700)]
    want, graphs = [], []
    for call, out, _ in steps:
        call()
        ctx.sync()
        want.append(out.clone())
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            call()
        graphs.append(g)
    for call, out, _ in larger:
        call()
    ctx.sync()
    filler = [torch.full((8 << 20,), 3.0, device="cuda") for _ in range(4)]  # (what was given back would be taken again)
    for _ in range(2):
        for g, (_, out, _), w in zip(graphs, steps, want):
            out.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            ctx.sync()
            assert torch.equal(out, w)
    assert all(bool((f == 3).all()) for f in filler)
    del graphs
    ctx.close()


def test_a_first_call_inside_a_capture_is_refused(ocr):
    maker, ctx = ocr.Context(0), ocr.Context(0)
    _, out, (cache, q, ps) = attend(ocr, maker, 3)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(ctx.stream())):
        with pytest.raises(ocr.OcrError, match="before capturing"):
            ocr.op_attention_window(ctx, cache, q, out, ps, 0.09)
    ocr.op_attention_window(ctx, cache, q, out, ps, 0.09)
    ctx.sync()
    assert out.any()
    del g
    ctx.close()
    maker.close()


# ---- after an error ----
class CtxHead(C.Structure):
    """the first fields of the context (csrc/ctx.h)"""
    _fields_ = [("refs", C.c_int), ("device", C.c_int), ("stream", C.c_void_p), ("num_sms", C.c_int), ("pdl", C.c_bool),
                ("d_err", C.c_void_p), ("mem", C.c_uint64 * 3), ("op_scratch", C.c_void_p),
                ("op_scratch_bytes", C.c_size_t), ("kv_work", C.c_void_p)]


class Ints:
    """device memory as torch.as_tensor takes it"""

    def __init__(self, address, n):
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="<i4", data=(address, False), version=3)


@pytest.mark.parametrize("T", [1, 8, 100])
def test_tickets_are_set_back_after_any_error(ocr, T):
    """A wait that runs out leaves tickets counted; the error flag keeps the first code, here a position's, so the code
    alone does not tell. (The tickets are set by the test in the place of the wait.)"""
    ctx = ocr.Context(0)
    call, out, (cache, q, ps) = attend(ocr, ctx, T, keys=6000)  # (two pairs over many CTAs)
    call()
    ctx.sync()
    want = out.clone()
    head = C.cast(ctx.h, C.POINTER(CtxHead)).contents
    assert head.device == 0 and head.stream == ctx.stream() and head.kv_work
    tickets = torch.as_tensor(Ints(head.kv_work, 1024), device="cuda")
    assert not tickets.any()
    tickets.fill_(1)
    torch.cuda.synchronize()
    ocr.op_attention_window(ctx, cache, q, torch.zeros_like(q), i32([6001]), 0.09)
    with pytest.raises(ocr.OcrError, match="position outside"):
        ctx.sync()
    ctx.sync()
    assert not tickets.any()
    out.zero_()
    torch.cuda.synchronize()
    call()
    ctx.sync()
    assert torch.equal(out, want)
    ctx.close()


# ---- the last rows of a cache ----
@pytest.mark.parametrize("T", [8, 40])
@pytest.mark.parametrize("kind", TYPES)
def test_a_ragged_step_at_the_end_of_the_cache(ocr, ctx, kind, T):
    """trees of fewer drafts than the call's rows, the longest slot's last draft in the cache's last row: written,
    attended, and the accepted rows moved"""
    n_kv, d, n_rows = 2, 128, 100
    pos, n = [n_rows - 5, 11, n_rows - T], [5, T, T]
    paths = [[0, 2, 4], list(range(0, T, 2)), [1, T - 1]]
    cache = make_cache(ocr, kind, 3, n_kv, n_rows, d)
    k, v = sequences(31, 3, n_rows + T, n_kv, d)
    put(ocr, ctx, cache, k[:, :n_rows], v[:, :n_rows], [0] * 3, n=pos)
    parents = [tree(7 + b, T) for b in range(3)]
    kd, vd = (torch.from_numpy(np.stack([x[b, pos[b]:pos[b] + T] for b in range(3)])).cuda() for x in (k, v))
    q = torch.from_numpy(np.random.default_rng(5).standard_normal((3, T, 4, d), dtype=np.float32)).cuda()
    out, ps, ns, par = torch.zeros_like(q), i32(pos), i32(n), i32(parents)
    torch.cuda.synchronize()
    ocr.op_kv_write(ctx, cache, kd, vd, ps, ns)
    ocr.op_attention_tree(ctx, cache, q, out, ps, par, 0.09, ns)
    ctx.sync()
    for b in range(3):
        m = n[b]
        kb, vb = (torch.from_numpy(P.held(x[b, :pos[b] + m], kind)).double().transpose(0, 1) for x in (k, v))
        want = P.attend(q[b, :m].double().cpu(), kb, vb, pos[b], 0.09, parent=parents[b][:m])
        assert float((out[b, :m].double().cpu() - want).abs().max() / vb.abs().max()) <= TOL["f32"]
    was = [t.clone() for t in cache._keep if t is not None]
    path, kept = i32([p + [0] * (T - len(p)) for p in paths]), i32([len(p) for p in paths])
    torch.cuda.synchronize()
    ocr.op_kv_keep(ctx, [cache], ps, path, kept)
    ctx.sync()
    for now, old in zip([t for t in cache._keep if t is not None], was):
        want = old.clone()
        for b in range(3):
            for i, j in enumerate(paths[b]):
                want[b, :, pos[b] + i] = old[b, :, pos[b] + j]
        assert torch.equal(now, want)


@pytest.mark.parametrize("ring", [False, True])
def test_a_path_past_the_end_is_flagged(ocr, ctx, ring):
    """the slot concerned is left alone, the other served"""
    end = 0x7fffffff if ring else 50
    cache = make_cache(ocr, "q8_0", 2, 1, 50, 64, **(dict(window=20, sinks=2, ring=True) if ring else {}))
    for t in cache._keep:
        t.copy_(torch.arange(t.numel(), device="cuda").view(t.shape) % 100)
    was = [t.clone() for t in cache._keep]
    path, kept, ps = i32([[0, 3, 6, 0, 0, 0, 0, 0], [1, 2, 0, 0, 0, 0, 0, 0]]), i32([3, 2]), i32([end - 6, 5])
    torch.cuda.synchronize()
    ocr.op_kv_keep(ctx, [cache], ps, path, kept)
    with pytest.raises(ocr.OcrError, match="position outside"):
        ctx.sync()
    ps2 = i32([end - 7, -1])
    torch.cuda.synchronize()
    for t, old in zip(cache._keep, was):
        assert torch.equal(t[0], old[0]) and torch.equal(t[1, :, 5:7], old[1, :, 6:8])
    ocr.op_kv_keep(ctx, [cache], ps2, path, kept)  # (a position less: its last row is the cache's last)
    ctx.sync()

    def row(p):
        return P.row_of(p, 50, 2, ring)

    for t, old in zip(cache._keep, was):
        for i, j in enumerate((0, 3, 6)):
            assert torch.equal(t[0, :, row(end - 7 + i)], old[0, :, row(end - 7 + j)])


@pytest.mark.parametrize("kind", TYPES)
def test_a_tight_ring_is_read_at_once(ocr, ctx, kind):
    """n_rows = sinks + window takes one row a call; a read overwrites nothing and takes all that it holds"""
    n_kv, d, window, sinks, total = 2, 64, 24, 3, 70
    cache = make_cache(ocr, kind, 1, n_kv, window + sinks, d, window=window, sinks=sinks, ring=True)
    k, v = sequences(12, 1, total, n_kv, d)
    put(ocr, ctx, cache, k, v, [0], chunk=1)
    for first, m in ((total - window, window), (0, sinks)):
        back = [torch.zeros(1, m, n_kv, d, device="cuda") for _ in "kv"]
        ps = i32([first])
        torch.cuda.synchronize()
        ocr.op_kv_read(ctx, cache, *back, ps)
        ctx.sync()
        for x, got in zip((k, v), back):
            np.testing.assert_array_equal(got.cpu().numpy(), P.held(x[:, first:first + m], kind))
    many = torch.zeros(1, window + sinks + 1, n_kv, d, device="cuda")
    with pytest.raises(ocr.OcrError, match="more than the cache"):
        ocr.op_kv_read(ctx, cache, many, many, ps)
    with pytest.raises(ocr.OcrError, match="more than the cache"):
        ocr.op_kv_write(ctx, cache, back[0][:, :2], back[1][:, :2], ps)


def test_more_tiles_than_32_bits_count_are_refused(ocr, ctx):
    """4096 row blocks x 1000 kv heads x 525 key blocks of one slot are more than 2^31. The rows are one vector, seen
    from everywhere."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("not enough memory")
    x = torch.zeros(1, 1, 1, 64, dtype=torch.float16, device="cuda")
    q, ps = x.expand(1, 65536, 8000, 64), i32([0])
    cache = make_cache(ocr, "q4_0", 1, 1000, 67200, 64)
    with pytest.raises(ocr.OcrError, match="more than one launch"):
        ocr.op_attention_window(ctx, cache, q, q, ps, 0.1)
    ctx.sync()


# ---- numbers far apart ----
def by_block(got, want, v, kind):
    """the largest error in each block of 32 dims, in units of the block's largest |value|"""
    top = np.abs(P.held(v, kind)).reshape(-1, v.shape[-1] // 32, 32).max((0, 2))
    err = (got - want).abs().reshape(-1, v.shape[-1] // 32, 32).amax((0, 2)).numpy()
    return err / top


@pytest.mark.parametrize("T", [1, 8, 130, 700])  # whole numbers, warp-level products, tcgen05 in parts and whole
@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", TYPES)
def test_values_whose_blocks_differ_along_d(ocr, ctx, kind, d, item, T):
    """blocks of 32 dims 2^20 apart in size: an output's error is bounded by its own block's values (the weights' errors
    are the same for every dim), not by the largest block's"""
    held = {}

    def change(k, v):
        v *= np.exp2(np.repeat(np.linspace(-9, 11, d // 32), 32)).astype(np.float32)
        if item == "f16":
            v[:] = v.astype(np.float16)
        held["v"] = v

    call, want, _ = case(ocr, ctx, kind, item, (1, 2, 2, d, T, [900], 0, 0, False, False), change=change)
    err = by_block(call(), want, held["v"], kind)
    assert err.max() <= TOL[item], err


@pytest.mark.parametrize("T", [1, 8, 130, 700])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
def test_single_values_far_above_the_others(ocr, ctx, kind, window, T):
    """a few positions whose first block is 2^20 (q8_0) times the others', at the start, inside and at the end: the other
    blocks keep their own accuracy, whatever tile the large one lies in"""
    d, held = 128, {}

    def change(k, v):
        v *= np.float32(2.0 ** -4)
        for j in (3, 290, 700, 890):
            v[:, j, :, :32] *= np.float32(2.0 ** (20 if kind == "q8_0" else 16))
        held["v"] = v

    call, want, _ = case(ocr, ctx, kind, "f32", (1, 2, 2, d, T, [900], window, 4 if window else 0, False, False), change=change)
    err = by_block(call(), want, held["v"], kind)
    assert err.max() <= TOL["f32"], err


@pytest.mark.parametrize("G", [2, 8, 64])  # whole numbers, warp-level products, tcgen05
@pytest.mark.parametrize("kind", TYPES)
def test_weights_of_f16_rows_are_rounded_once(ocr, ctx, kind, G):
    """One position far above the others with values of zero, the others all alike: their weights' rounding errors are the
    same and do not average out. One rounding to f16 is 2^-11 of the output, the output's own half a unit in its last
    place; scores and sums in f32 add less than 10^-5."""
    n_slot, n_kv, d, n = 12, 8, 128, 33
    g = np.random.default_rng(17)
    k, v = np.zeros((n_slot, n, n_kv, d), np.float32), np.zeros((n_slot, n, n_kv, d), np.float32)
    k[:, 0, :, 0] = 4.0
    v[:, 1:] = np.repeat(g.uniform(0.3, 3, (n_slot, 1, n_kv, d // 32)), 32, -1)
    q = np.zeros((n_slot, 1, n_kv * G, d), np.float16)
    q[..., 0] = g.uniform(0.2, 4, q.shape[:3])
    cache = make_cache(ocr, kind, n_slot, n_kv, n, d)
    put(ocr, ctx, cache, k, v, [0] * n_slot)
    qd = torch.from_numpy(q).cuda()
    out, ps = torch.zeros_like(qd), i32([n - 1] * n_slot)
    torch.cuda.synchronize()
    ocr.op_attention_window(ctx, cache, qd, out, ps, 0.5)
    ctx.sync()
    got = out.double().cpu().numpy()
    for b in range(n_slot):
        kb, vb = (torch.from_numpy(P.held(x[b], kind)).double().transpose(0, 1) for x in (k, v))
        want = P.attend(torch.from_numpy(q[b]).double(), kb, vb, n - 1, 0.5).numpy()
        half_ulp = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2
        assert (np.abs(got[b] - want) <= (2.0 ** -11 + 1e-5) * np.abs(want) + half_ulp).all()


@pytest.mark.parametrize("T,G", [(1, 2), (3, 2), (1, 12), (8, 4), (130, 2), (700, 2)])
@pytest.mark.parametrize("item", ["f32", "f16"])
def test_infinite_keys(ocr, ctx, item, T, G):
    """an infinite value in an f16 key, written as one or as a finite f32 beyond f16's range: a row whose query has the
    other sign there gives the key no weight; one of the same sign has no finite output"""
    def change(k, v):
        k[0, 40, 0, 7] = np.inf
        k[0, 41, 0, 9] = -np.inf
        k[0, 300, 0, 7] = 1e5 if item == "f32" else np.inf
        k[0, 401, 0, 70] = -1e30 if item == "f32" else -np.inf

    with np.errstate(over="ignore"):
        call, want, top = case(ocr, ctx, "f16", item, (1, 2, G, 128, T, [401], 0, 0, False, False), change=change)
    got = call()
    fine = torch.isfinite(want)
    assert 0.05 < float(fine[..., 0].double().mean()) < 0.95
    assert float((got - want)[fine].abs().max()) / top <= TOL[item]
    assert not torch.isfinite(got[~fine]).any()


@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("kind", TYPES)
def test_sums_over_a_million_keys(ocr, ctx, kind, item):
    """Rows on the tensor cores, every triple in one CTA, values of one size: the output is the value. A sum in TMEM may lose
    10^-7 of itself at each product; it is moved out after 64 (f32 rows) or 256 (f16 rows) of them: 6.4 10^-6, 2.6 10^-5.
    With the sum of the weights, 10^-5 and 5 10^-5 are allowed, beside half a unit of the output in f16."""
    n, T, G, d = 1_000_000, 148, 128, 64
    cache = make_cache(ocr, kind, 1, 1, n + T, d)
    g = torch.Generator(device="cuda").manual_seed(3)
    for a in range(0, n + T, 1 << 17):
        m = min(1 << 17, n + T - a)
        k = torch.randn(1, m, 1, d, device="cuda", generator=g)
        ps = i32([a])
        torch.cuda.synchronize()
        ocr.op_kv_write(ctx, cache, k, torch.ones_like(k), ps)
        ctx.sync()
    q = torch.randn(1, T, G, d, device="cuda", generator=g).to(ITEM[item])
    out, ps = torch.zeros_like(q), i32([n])
    torch.cuda.synchronize()
    ocr.op_attention_window(ctx, cache, q, out, ps, 0.125)
    ctx.sync()
    one = float(P.held(np.ones((1, 32), np.float32), kind)[0, 0])  # (1, or a little less: half a unit is 2^-12)
    assert one <= 1
    assert float((out.double() - one).abs().max()) <= (2.0 ** -12 + 5e-5 if item == "f16" else 1e-5)


# ---- shapes between the kernels' ordinary ones ----
BETWEEN = [  # (as test_gpu_kv.SHAPES) two rows of one head: whole numbers over quants
    (2, 2, 1, 128, 2, [300, 5], 0, 0, False, False),
    (2, 2, 1, 64, 2, [200, 77], 40, 3, False, False),
    (1, 1, 1, 128, 2, [500], 33, 4, True, False),
    (3, 2, 1, 128, 2, [260, -1, 0], 0, 0, False, True),
    (2, 1, 1, 64, 2, [400, 90], 50, 5, False, True),
    (1, 8, 1, 128, 2, [6000], 0, 0, False, False),
    # five to eight pairs of several rows: one warp to a team, hi and lo in products of their own
    (2, 2, 2, 128, 3, [310, 9], 0, 0, False, False),
    (1, 2, 1, 64, 7, [150], 20, 2, False, False),
    (2, 1, 4, 128, 2, [270, 31], 64, 4, True, False),
    (2, 2, 1, 128, 6, [199, 0], 0, 0, False, True),
    (1, 1, 1, 64, 8, [333], 30, 6, False, True),
    (1, 8, 2, 128, 4, [5000], 0, 0, False, False),
]


@pytest.mark.parametrize("shape", BETWEEN, ids=lambda s: "-".join(map(str, s)).replace(" ", ""))
@pytest.mark.parametrize("item", ["f32", "f16"])
@pytest.mark.parametrize("kind", TYPES)
def test_shapes_between(ocr, ctx, kind, item, shape):
    call, want, top = case(ocr, ctx, kind, item, shape)
    got = call()
    assert float((got - want).abs().max()) / top <= TOL[item]
    assert torch.equal(got, call())


@pytest.mark.parametrize("shape", [s for s in BETWEEN if max(s[5]) < 1000], ids=lambda s: "-".join(map(str, s)).replace(" ", ""))
@pytest.mark.parametrize("kind", TYPES)
def test_what_rows_of_these_shapes_do_not_see(ocr, ctx, kind, shape):
    common.test_what_a_row_does_not_see_has_no_part(ocr, ctx, kind, shape)


@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("kind", TYPES)
def test_a_tree_of_one_draft(ocr, ctx, kind, G):
    """it sees what a row sees, and its parent is looked at as in any tree"""
    cache = make_cache(ocr, kind, 2, 1, 300, 128, window=100, sinks=3)
    k, v = sequences(44, 2, 300, 1, 128)
    put(ocr, ctx, cache, k, v, [0, 0])
    q = torch.randn(2, 1, G, 128, device="cuda")
    out, want, ps = torch.zeros_like(q), torch.zeros_like(q), i32([299, 50])
    good, bad = i32([[-1], [-1]]), i32([[-1], [0]])
    torch.cuda.synchronize()
    ocr.op_attention_window(ctx, cache, q, want, ps, 0.09)
    ocr.op_attention_tree(ctx, cache, q, out, ps, good, 0.09)
    ctx.sync()
    assert float((out - want).abs().max()) <= TOL["f32"] * float(np.abs(P.held(v, kind)).max())
    ocr.op_attention_tree(ctx, cache, q, out, ps, bad, 0.09)
    with pytest.raises(ocr.OcrError, match="index outside"):
        ctx.sync()
