"""The cases that the quantised KV cache and its attention are measured at, and the operators' plain forms.

Three operators over one layer's KV cache, of n_slot sequences, whose rows are f16, q8_0 or q4_0:

  store   rows of keys and values are quantised into the cache as they are written, and read back as values;
  attend  rows of queries attend the cache: causal, within a sliding window, the first `sinks` positions always
          visible; from one row (a decode step) to a prompt's rows; in a ring cache the rows of positions that left
          the window are written again;
  tree    a step of drafted tokens: the drafts' keys and values are written after the committed rows, every draft
          attends the committed rows and its own ancestors, and the rows of the accepted path are moved together.

The cache's memory, which both forms read and write (row r of position p: p itself, or in a ring cache
sinks + (p - sinks) % (n_rows - sinks) for p >= sinks):
  f16   k, v [n_slot][n_kv][n_rows][d] f16
  q8_0  k, v [n_slot][n_kv][n_rows][d] int8, scales [n_slot][n_kv][n_rows][d / 32] f16: value = q * scale
  q4_0  k, v [n_slot][n_kv][n_rows][d / 2] uint8, scales as above: byte j of a block of 16 holds value j in its low
        nibble and value j + 16 in its high one; value = (nibble - 8) * scale
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
BLOCK = 32
DTYPE = {"f32": torch.float32, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step's new row of each of a full batch: the batched session's 32 slots, 8 kv heads of 128
        dict(name="store 32 x 1 q8_0", op="store", type="q8_0", rows_type="f32", slots=32, n_kv=8, d=128, rows=1,
             keys=3584, n_rows=4096, window=0, sinks=0, ring=False),
        # one page's prompt (2200 image rows and its ids) into a 4-bit cache
        dict(name="store 1 x 2214 q4_0", op="store", type="q4_0", rows_type="f32", slots=1, n_kv=8, d=128, rows=2214,
             keys=0, n_rows=4096, window=0, sinks=0, ring=False),
        # a whole batch's prompts
        dict(name="store 32 x 2214 q8_0", op="store", type="q8_0", rows_type="f32", slots=32, n_kv=8, d=128,
             rows=2214, keys=0, n_rows=4096, window=0, sinks=0, ring=False),
        # one page's decode step: one slot, one row, the smallest call, where latency counts
        dict(name="attend 1 x 1 q8_0", op="attend", type="q8_0", rows_type="f32", slots=1, n_head=16, n_kv=8, d=128,
             rows=1, keys=2303, n_rows=4096, window=0, sinks=0, ring=False),
        # a batch's decode step at ragged lengths: bandwidth counts
        dict(name="attend 32 x 1 q8_0", op="attend", type="q8_0", rows_type="f32", slots=32, n_head=16, n_kv=8, d=128,
             rows=1, keys=4095, n_rows=4096, window=0, sinks=0, ring=False),
        # the same far beyond the cache's rows: a ring of the last 1024 positions and four first ones, 4-bit
        dict(name="attend 32 x 1 q4_0 ring", op="attend", type="q4_0", rows_type="f32", slots=32, n_head=16, n_kv=8,
             d=128, rows=1, keys=40000, n_rows=1040, window=1024, sinks=4, ring=True),
        # a prompt's rows, each seeing the last 512 positions and four first ones
        dict(name="attend 1 x 2214 q8_0 window", op="attend", type="q8_0", rows_type="f32", slots=1, n_head=16, n_kv=8,
             d=128, rows=2214, keys=0, n_rows=4096, window=512, sinks=4, ring=False),
        # the next 512 rows of four long documents: f16 rows and cache, heads of 64, the largest call
        dict(name="attend 4 x 512 f16 long", op="attend", type="f16", rows_type="f16", slots=4, n_head=16, n_kv=4,
             d=64, rows=512, keys=16384, n_rows=17000, window=0, sinks=0, ring=False),
        # a chunk of rows in f32 over an f16 cache, as a prompt continues
        dict(name="attend 2 x 333 f16", op="attend", type="f16", rows_type="f32", slots=2, n_head=16, n_kv=8, d=128,
             rows=333, keys=1881, n_rows=2500, window=0, sinks=0, ring=False),
        # drafts for one page: 16 tokens in a tree
        dict(name="tree 1 x 16 q8_0", op="tree", type="q8_0", rows_type="f32", slots=1, n_head=16, n_kv=8, d=128,
             rows=16, keys=2303, n_rows=4096, window=0, sinks=0, ring=False),
        # drafts for a batch, ragged lengths
        dict(name="tree 32 x 8 q8_0", op="tree", type="q8_0", rows_type="f32", slots=32, n_head=16, n_kv=8, d=128,
             rows=8, keys=4080, n_rows=4096, window=0, sinks=0, ring=False),
        # wide trees over long windows, four query heads to a key head
        dict(name="tree 8 x 61 q4_0 window", op="tree", type="q4_0", rows_type="f16", slots=8, n_head=32, n_kv=8,
             d=128, rows=61, keys=12001, n_rows=12100, window=8192, sinks=16, ring=False),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    cap = {}
    for c in listed():
        w = work(c)
        cap[c["op"]] = max(cap.get(c["op"], 0.0), w["bytes"] / 6.5e12 + w["flops"] / 1e15)
    op = rng.choice(["store", "attend", "attend", "tree"])
    while True:
        n_kv = rng.choice([1, 2, 4, 8])
        c = dict(op=op, type=rng.choice(["f16", "q8_0", "q4_0"]), rows_type=rng.choice(["f32", "f32", "f16"]),
                 slots=_log(rng, 1, 64), n_kv=n_kv, d=rng.choice([64, 128, 128]),
                 keys=_log(rng, 16, 40000))
        if op != "store":
            c["n_head"] = n_kv * rng.choice([1, 2, 2, 4, 8])
        many = op == "attend" and rng.random() < 0.5
        c["rows"] = _log(rng, 1, 2300) if op == "store" else _log(rng, 2, 64) if op == "tree" else \
            _log(rng, 2, 2300) if many else 1
        c["window"], c["sinks"], c["ring"] = 0, 0, False
        if rng.random() < 0.5:
            c["window"], c["sinks"] = _log(rng, 64, 4096), rng.choice([0, 1, 4, 16, 64])
            c["ring"] = rng.random() < 0.5
        if c["ring"]:
            c["n_rows"] = c["sinks"] + c["window"] + c["rows"] - 1 + rng.randint(0, 40)
        else:
            c["n_rows"] = c["keys"] + c["rows"] + rng.randint(0, 100)
        held = c["slots"] * n_kv * c["n_rows"] * c["d"]  # the plain form holds the cache in 32 bits
        scores = c["slots"] * c.get("n_head", 0) * c["rows"] * c["n_rows"]
        w = work(c)
        if held <= 5e8 and scores <= 6e8 and w["bytes"] / 6.5e12 + w["flops"] / 1e15 <= cap[op]:
            return c


def _lengths(case):
    """committed positions of each slot: one slot has `keys`, a batch from half of it to all of it, in no order"""
    n, keys = case["slots"], case["keys"]
    if n == 1:
        return [keys]
    step = next(p for p in (13, 17, 19, 23, 29) if math.gcd(p, n) == 1)
    return [keys - keys // 2 + (keys // 2) * ((i * step) % n) // (n - 1) for i in range(n)]


def _parents(case):
    """a tree of drafts for each slot: parent[i] < i, -1 for a child of the last committed token"""
    rng = random.Random(case["rows"] * 1009 + case["slots"])
    return [[rng.randint(max(-1, i - 1 - rng.choice([0, 1, 4, 16])), i - 1) if i else -1 for i in range(case["rows"])]
            for _ in range(case["slots"])]


def _path(parent):
    """the drafts from the root to the last one"""
    path, i = [], len(parent) - 1
    while i >= 0:
        path.append(i)
        i = parent[i]
    return path[::-1]


def _row_bytes(case):
    d = case["d"]
    return {"f16": 2 * d, "q8_0": d + d // 16, "q4_0": d // 2 + d // 16}[case["type"]]


def _visible(case):
    """of all slots: the positions that any row sees, and (row, position) pairs that are seen"""
    held = pairs = 0
    w, s, T = case["window"], case["sinks"], case["rows"]
    trees = _parents(case) if case["op"] == "tree" else None
    for b, n in enumerate(_lengths(case)):
        depth = None
        if trees:
            depth = []
            for p in trees[b]:
                depth.append(0 if p < 0 else depth[p] + 1)
        lo = max(0, n - w + 1) if w else 0  # the first position in the first row's window
        held += n + T - lo + min(s, lo)
        for t in range(T):
            at = n + (depth[t] if trees else t)
            first = max(0, at - w + 1) if w else 0
            pairs += at + 1 - first + min(s, first)
    return held, pairs


def work(case):
    rows = case["slots"] * case["rows"]
    item = 4 if case["rows_type"] == "f32" else 2
    kv_row = 2 * case["n_kv"] * _row_bytes(case)
    kv_in = 2 * case["n_kv"] * case["d"] * item
    if case["op"] == "store":  # rows in, the cache written and read, rows out
        return {"bytes": rows * (2 * kv_in + 2 * kv_row), "flops": 6 * rows * 2 * case["n_kv"] * case["d"]}
    held, pairs = _visible(case)
    out = {"bytes": held * kv_row + 2 * rows * case["n_head"] * case["d"] * item,
           "flops": 4 * pairs * case["n_head"] * case["d"]}
    if case["op"] == "tree":  # the drafts in and written, the accepted rows moved and read back
        kept = sum(len(_path(p)) for p in _parents(case))
        out["bytes"] += rows * (kv_in + kv_row) + kept * (3 * kv_row + kv_in)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------------------------------------------------
def _empty(case, dev):
    lead = (case["slots"], case["n_kv"], case["n_rows"])
    width, dtype = {"f16": (case["d"], torch.float16), "q8_0": (case["d"], torch.int8),
                    "q4_0": (case["d"] // 2, torch.uint8)}[case["type"]]
    c = {n: torch.zeros(*lead, width, dtype=dtype, device=dev) for n in ("k", "v")}
    if case["type"] != "f16":
        c.update({n: torch.zeros(*lead, case["d"] // BLOCK, dtype=torch.float16, device=dev)
                  for n in ("k_scale", "v_scale")})
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    B, T, n_kv, d = case["slots"], case["rows"], case["n_kv"], case["d"]
    n_head = case.get("n_head", 0)
    item = DTYPE[case["rows_type"]]
    # keys as after the per-head norm, with a few large channels; values of mixed sizes; the new rows stand together
    # as [q heads | k heads | v heads], as the projection leaves them
    chan = 1 + 3 * (torch.rand(n_kv, d, device=dev, generator=g) < 0.04)
    qkv = torch.randn(B, T, n_head + 2 * n_kv, d, device=dev, generator=g)
    qkv[:, :, :n_head] *= 1.5
    qkv[:, :, n_head:n_head + n_kv] *= chan
    qkv[:, :, n_head + n_kv:] *= 0.7
    qkv = qkv.to(item)
    # what the cache holds: every row, those past a slot's length too (they are a former page's)
    cache = _empty(case, dev)
    for b in range(B):
        k = torch.randn(n_kv, case["n_rows"], d, device=dev, generator=g) * chan[:, None]
        v = torch.randn(n_kv, case["n_rows"], d, device=dev, generator=g) * 0.7
        for n, x in (("k", k), ("v", v)):
            q, scale = _quantise(x, case["type"])
            cache[n][b] = q
            if scale is not None:
                cache[n + "_scale"][b] = scale
    s = dict(case=case, qkv=qkv, cache=cache, scale=1.0 / math.sqrt(d),
             q=qkv[:, :, :n_head], k=qkv[:, :, n_head:n_head + n_kv], v=qkv[:, :, n_head + n_kv:],
             pos=torch.tensor(_lengths(case), dtype=torch.int32, device=dev))
    if n_head:
        s["out"] = torch.zeros(B, T, n_head, d, dtype=item, device=dev)
    if case["op"] == "tree":
        trees = _parents(case)
        paths = [_path(p) for p in trees]
        s["longest"] = max(map(len, paths))
        s["parent"] = torch.tensor(trees, dtype=torch.int32, device=dev)
        s["path"] = torch.tensor([p + [0] * (T - len(p)) for p in paths], dtype=torch.int32, device=dev)
        s["kept"] = torch.tensor(list(map(len, paths)), dtype=torch.int32, device=dev)
    if case["op"] != "attend":
        n = s.get("longest", T)
        s["back"] = [torch.zeros(B, n, n_kv, d, dtype=item, device=dev) for _ in "kv"]
    if own:  # the view of the cache's memory that a program keeps beside it
        s["view"] = _ocr().KvCache(case["type"], **cache, d_head=d, window=case["window"], sinks=case["sinks"],
                                   ring=case["ring"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: elementary operations, in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _quantise(x, kind):
    """rows of f32 values → what the cache holds of them"""
    if kind == "f16":
        return x.to(torch.float16), None
    xb = x.float().unflatten(-1, (-1, BLOCK))
    mag = xb.abs()
    amax = mag.amax(-1, keepdim=True)
    if kind == "q8_0":
        step = amax / torch.full_like(amax, 127.0)  # (a division, not a product with 1 / 127)
    else:  # the first value of the largest magnitude becomes -8
        place = torch.arange(BLOCK, device=x.device).expand_as(mag)
        first = torch.where(mag == amax, place, BLOCK).amin(-1, keepdim=True)
        step = xb.gather(-1, first) / -8.0
    scale = step.to(torch.float16)
    y = xb * torch.where(step != 0, 1.0 / step, 0.0)
    y = torch.where(scale != 0, y, 0.0)
    if kind == "q8_0":  # to the nearest, halves away from zero
        a = y.abs()
        low = a.floor()
        q = torch.copysign(low + ((a - low) >= 0.5), y).to(torch.int8).flatten(-2)
    else:
        n = (y + 8.5).floor().clamp(0, 15).to(torch.uint8)
        q = (n[..., :16] | (n[..., 16:] << 4)).flatten(-2)
    return q, scale.squeeze(-1)


def _values(q, scale, kind):
    if kind == "f16":
        return q.float()
    if kind == "q4_0":
        b = q.unflatten(-1, (-1, BLOCK // 2))
        n = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    else:
        n = q.unflatten(-1, (-1, BLOCK)).float()
    return (n * scale.float()[..., None]).flatten(-2)


def _row(case, p):
    s = case["sinks"]
    return torch.where(p < s, p, s + (p - s) % (case["n_rows"] - s)) if case["ring"] else p


def _places(s, first, n):
    """indices (slot, head, row) of positions first … first + n - 1 of every slot"""
    case = s["case"]
    rows = _row(case, first[:, None].long() + torch.arange(n, device=first.device))
    b = torch.arange(case["slots"], device=first.device)
    return b[:, None, None], torch.arange(case["n_kv"], device=first.device)[None, None], rows[:, :, None]


def _write(s):
    at = _places(s, s["pos"], s["case"]["rows"])
    for n in ("k", "v"):
        q, scale = _quantise(s[n], s["case"]["type"])
        s["cache"][n][at] = q
        if scale is not None:
            s["cache"][n + "_scale"][at] = scale


def _read(s, n_rows):
    at = _places(s, s["pos"], n_rows)
    c, kind = s["cache"], s["case"]["type"]
    return [_values(c[n][at], c[n + "_scale"][at] if kind != "f16" else None, kind).to(s[n].dtype) for n in ("k", "v")]


def _attend(s, tree):
    case, c, dev = s["case"], s["cache"], s["q"].device
    B, T, H, n_kv, d = case["slots"], case["rows"], case["n_head"], case["n_kv"], case["d"]
    end = int(max(_lengths(case))) + T
    # the position that each row of the cache holds, once all rows of this call are written
    j = torch.arange(min(case["n_rows"], end), device=dev)
    last = s["pos"].long()[:, None] + T - 1
    kp = j.expand(B, -1)
    if case["ring"]:
        sink, ring = case["sinks"], case["n_rows"] - case["sinks"]
        held = last - ((last - sink) - (j - sink)) % ring
        kp = torch.where(j < sink, kp, torch.where(held >= sink, held, last + 1))
    pos = s["pos"].long()[:, None]
    at = torch.arange(T, device=dev).expand(B, T)
    seen = None
    if tree:  # each draft's ancestors, itself among them: sums of paths of every length, scaled to stay finite
        link = s["parent"].long()[:, :, None] == torch.arange(T, device=dev)
        seen = torch.linalg.matrix_power((torch.eye(T, device=dev) + link) / 2, T) > 0
        at = seen.sum(-1) - 1
    qp = (pos + at)[:, :, None]
    kp = kp[:, None, :]
    own_rows = kp - pos[:, :, None]  # >= 0: the index of one of this call's rows
    if tree:
        depth = torch.gather(at[:, None, :].expand(B, T, T), 2, own_rows.clamp(0, T - 1).expand(B, T, -1))
        among = torch.gather(seen, 2, own_rows.clamp(0, T - 1).expand(B, T, -1))
        where = torch.where(own_rows >= 0, pos[:, :, None] + depth, kp)
        mask = torch.where(own_rows >= 0, among & (own_rows < T), True)
    else:
        where, mask = kp, kp <= qp
    if case["window"]:
        mask = mask & ((where > qp - case["window"]) | (where < case["sinks"]))
    n = j.numel()
    k, v = (_values(c[x][:, :, :n], c[x + "_scale"][:, :, :n] if case["type"] != "f16" else None, case["type"])
            for x in ("k", "v"))
    q = s["q"].float().reshape(B, T, n_kv, H // n_kv, d).permute(0, 2, 3, 1, 4).reshape(B, n_kv, -1, d)
    x = torch.matmul(q, k.transpose(-1, -2)).view(B, n_kv, H // n_kv, T, n) * s["scale"]
    x = x.masked_fill(~mask[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, n_kv, -1, n), v).view(B, n_kv, H // n_kv, T, d)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, d).to(s["q"].dtype)


def _keep(s):
    """the accepted drafts' rows move to the committed rows' end"""
    case, c = s["case"], s["cache"]
    n = s["longest"]
    b, h, src = _places(s, s["pos"], case["rows"])
    i = torch.arange(n, device=src.device)
    # past a slot's own path: rows stay where they are
    take = torch.where(i < s["kept"][:, None], s["path"][:, :n].long(), i)
    src, dst = torch.gather(src, 1, take[:, :, None]), src[:, :n]
    for x in c.values():
        x[b, h, dst] = x[b, h, src]


def _plain(s):
    op = s["case"]["op"]
    if op == "store":
        _write(s)
        return _read(s, s["case"]["rows"])
    if op == "attend":
        return _attend(s, False)
    _write(s)
    out = _attend(s, True)
    _keep(s)
    k, v = _read(s, s["longest"])
    live = (torch.arange(s["longest"], device=k.device) < s["kept"][:, None])[:, :, None, None]
    return [out, torch.where(live, k, 0), torch.where(live, v, 0)]


# ---------------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------------
_lib = {}


def _ocr():
    if not _lib:
        sys.path.insert(0, str(ROOT / "historic-htr-ocr_b200"))
        import ocr_b200

        _lib["ocr"], _lib["ctx"] = ocr_b200, ocr_b200.Context(torch.cuda.current_device())
    return _lib["ocr"]


def _own(s):
    ocr, ctx = _ocr(), _lib["ctx"]
    op, view = s["case"]["op"], s["view"]
    if op == "store":
        ocr.op_kv_write(ctx, view, s["k"], s["v"], s["pos"])
        ocr.op_kv_read(ctx, view, s["back"][0], s["back"][1], s["pos"])
        return s["back"]
    if op == "attend":
        ocr.op_attention_window(ctx, view, s["q"], s["out"], s["pos"], s["scale"])
        return s["out"]
    ocr.op_kv_write(ctx, view, s["k"], s["v"], s["pos"])
    ocr.op_attention_tree(ctx, view, s["q"], s["out"], s["pos"], s["parent"], s["scale"])
    ocr.op_kv_keep(ctx, [view], s["pos"], s["path"], s["kept"])
    ocr.op_kv_read(ctx, view, s["back"][0], s["back"][1], s["pos"], n=s["kept"])
    return [s["out"]] + s["back"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits, row by row
# ---------------------------------------------------------------------------------------------------------------------
def _exact_block(x, kind):
    """x [..., 32] f64 → the values that the cache stands for"""
    big = x.abs().max(-1, keepdim=True).values
    if kind == "q8_0":
        step = big / 127
    else:
        i = (x.abs() == big).double().mul(torch.arange(32, 0, -1, device=x.device)).max(-1, keepdim=True).indices
        step = -torch.take_along_dim(x, i, -1) / 8
    held = step.half().double()
    y = torch.where(held != 0, x / step, 0.0)
    n = torch.sign(y) * (y.abs() + 0.5).floor() if kind == "q8_0" else ((y + 8.5).floor().clamp(0, 15) - 8)
    return n * held


def _exact_held(x, kind):
    if kind == "f16":
        return x.half().double()
    return _exact_block(x.double().reshape(-1, 32), kind).reshape(x.shape)


def _exact_cache(case, s, b, name):
    """the values of slot b's rows [n_kv][n_rows][d]"""
    x = s["cache"][name][b]
    if case["type"] == "f16":
        return x.double()
    scale = s["cache"][name + "_scale"][b].double().repeat_interleave(32, -1)
    if case["type"] == "q8_0":
        return x.double() * scale
    x = x.long().reshape(*x.shape[:-1], -1, 16)
    return (torch.stack([x % 16, x // 16], -2).reshape(scale.shape) - 8).double() * scale


def exact(case, seed):
    s = prepare(case, seed)
    op, T, kind = case["op"], case["rows"], case["type"]
    if op == "store":
        return [_exact_held(s[n], kind) for n in ("k", "v")]
    n_kv, H, d, w, sinks = case["n_kv"], case["n_head"], case["d"], case["window"], case["sinks"]
    out = torch.zeros(case["slots"], T, H, d, dtype=torch.float64, device=s["q"].device)
    trees = _parents(case)
    back = [torch.zeros(*x.shape, dtype=torch.float64, device=x.device) for x in s.get("back", [])]
    for b, n in enumerate(_lengths(case)):
        total = n + T
        rows = torch.arange(total, device=out.device)
        if case["ring"]:
            rows = torch.where(rows < sinks, rows, sinks + (rows - sinks) % (case["n_rows"] - sinks))
        k, v = (_exact_cache(case, s, b, x) for x in ("k", "v"))
        if op == "tree":
            new = [_exact_held(s[x][b], kind) for x in ("k", "v")]
            for x, y in zip((k, v), new):
                x[:, rows[n:]] = y.transpose(0, 1)
            path = _path(trees[b])
            for x, y in zip(back, new):
                x[b, :len(path)] = y[path]
            see = torch.zeros(T, total, dtype=torch.bool)
            depth = []
            for i, p in enumerate(trees[b]):
                depth.append(0 if p < 0 else depth[p] + 1)
                see[i, :n] = True
                if p >= 0:
                    see[i, n:] = see[p, n:]
                see[i, n + i] = True
            see, depth = see.to(out.device), torch.tensor(depth, device=out.device)
            place = torch.cat([torch.arange(n, device=out.device), n + depth])
            mine = n + depth
        else:
            place = torch.arange(total, device=out.device)
            mine = place[n:]
            see = place[None] <= mine[:, None]
        if w:
            see &= (mine[:, None] - place[None] < w) | (place[None] < sinks)
        cols = see.any(0).nonzero()[:, 0]  # (a ring's rows of positions that left every window hold others)
        see = see[:, cols]
        for h in range(H):
            kh, vh = (x[h // (H // n_kv), rows[cols]] for x in (k, v))
            e = (s["q"][b, :, h].double() @ kh.T) * s["scale"]
            p = torch.softmax(torch.where(see, e, -math.inf), -1)
            out[b, :, h] = p @ vh
    return out if op == "attend" else [out] + back
