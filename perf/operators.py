"""Workloads of the table lookup (``ops.embedding`` and its gradient) and of the gated scan along segments
(``ops.gated_scan``, ``ops.gated_scan_step``).

A case is one call as a model makes it; ``run`` computes it in plain torch operations (``own`` false) or through the
package (``own`` true).  Sizes: the buildings of this repository (8 graphs of 1,440 voxels, hidden widths 128 / 256,
7 program classes, 20 floor levels, variation batches of 1,048,576 voxels) and the generic ones of token models.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _lookup(name, op, dtype, tokens, vocab, width, skew=False, missing=False, ids="i64"):
    case = {"op": op, "dtype": dtype, "tokens": tokens, "vocab": vocab, "width": width, "skew": skew, "missing": missing,
            "ids": ids}
    return dict(case, name=name) if name else case


def _scan(name, op, dtype, rows, segments, width, layout="even", reverse=False, packed=False):
    case = {"op": op, "dtype": dtype, "rows": rows, "segments": segments, "width": width, "layout": layout, "reverse": reverse,
            "packed": packed}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one new token for each of eight requests that are being answered: nothing but latency
        _lookup("lookup-8-tokens-bf16", "lookup", "bf16", 8, 32000, 1024),
        # the floor level of every voxel of a batch of eight buildings, read from a learned position table
        _lookup("lookup-levels-f32", "lookup", "f32", 11520, 20, 128, ids="i32"),
        # a training step's tokens, frequent ones first as in text, over an ordinary vocabulary
        _lookup("lookup-train-text-bf16", "lookup_train", "bf16", 16384, 32000, 1024, skew=True),
        # a large vocabulary, an odd number of tokens, padding tokens among them
        _lookup("lookup-train-missing-f16", "lookup_train", "f16", 65537, 131071, 520, missing=True),
        # the program class of every voxel of a variation batch: a million rows into seven sums
        _lookup("lookup-train-classes-f32", "lookup_train", "f32", 1048576, 7, 128),
        # one step up for 50 stories whose states are kept between calls
        _scan("step-stories-f32", "step", "f32", 50, 50, 256),
        # the voxels of a batch of eight buildings, in scan order, without a gradient
        _scan("scan-buildings-f32", "scan", "f32", 11520, 8, 128),
        # the same in training, both halves of one projection, at the discriminator's width
        _scan("scan-train-buildings-f32", "scan_train", "f32", 11520, 8, 256, packed=True),
        # a training step over four sequences of ordinary length
        _scan("scan-train-text-bf16", "scan_train", "bf16", 16384, 4, 2048, packed=True),
        # ragged sequences, empty ones and single rows among them, rows behind the last, an odd width, backwards
        _scan("scan-train-ragged-f16", "scan_train", "f16", 100003, 301, 333, layout="ragged", reverse=True),
        # one building of a million voxels
        _scan("scan-million-f32", "scan", "f32", 1048576, 1, 128),
        # two long sequences in training
        _scan("scan-train-long-bf16", "scan_train", "bf16", 262144, 2, 512),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; one in two is odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, n | 1 if rng.random() < 0.5 else n))


def draw(rng):
    """Another case of the same ranges: 8 tokens to a million, 7 rows of table to 131,072, widths from 16 to 2,048,
    one sequence to hundreds; the elements of a case stay under those of the largest listed one (2^27)."""
    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["lookup", "lookup_train", "lookup_train", "step", "scan", "scan_train", "scan_train"])
    width = _spread(rng, 16, 2048)
    if rng.random() < 0.5:
        width = max(16, width // 16 * 16)
    if op in ("lookup", "lookup_train"):
        vocab = _spread(rng, 7, min(131072, (1 << 26) // width))
        tokens = _spread(rng, 8, min(1048576, (1 << 26) // width))
        return _lookup(None, op, dtype, tokens, vocab, width, skew=rng.random() < 0.5, missing=rng.random() < 0.3,
                       ids=rng.choice(["i64", "i32"]))
    if op == "step":
        n = _spread(rng, 1, 512)
        return _scan(None, op, dtype, n, n, width)
    rows = _spread(rng, 64, min(1048576, (1 << (27 if op == "scan" else 26)) // width))
    if rng.random() < 0.5:
        segments = _spread(rng, 1, max(1, min(512, rows // 8)))
        return _scan(None, op, dtype, rows, segments, width, layout="ragged", reverse=rng.random() < 0.5,
                     packed=rng.random() < 0.5)
    segments = _spread(rng, 1, max(1, min(64, rows // 64)))
    return _scan(None, op, dtype, rows // segments * segments, segments, width, reverse=rng.random() < 0.5,
                 packed=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _lookup_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    n, v, d, dt = case["tokens"], case["vocab"], case["width"], _DT[case["dtype"]]
    u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
    if case["skew"]:        # p(id) = log((id + 2) / (id + 1)) / log(vocab + 1): nearly 1 / rank, as in text
        ids = torch.exp(u * math.log(v + 1)).long() - 1
    else:
        ids = (u * v).long()
    ids.clamp_(0, v - 1)
    if case["missing"]:     # padding tokens
        ids[torch.rand(n, generator=gen, device=dev) < 0.0625] = -1
    weight = (torch.randn(v, d, generator=gen, device=dev) * 0.02).to(dt)
    st = {"case": case, "ids": ids if case["ids"] == "i64" else ids.int(), "weight": weight, "scale": math.sqrt(d)}
    if case["op"] == "lookup_train":
        st["weight"] = weight.requires_grad_(True)
        st["dout"] = (torch.randn(n, d, generator=gen, device=dev) * 0.01).to(dt)
    return st


def _segment_rows(case, gen_cpu):
    """Row pointer of the segments, as a list."""
    n, s = case["rows"], case["segments"]
    if case["layout"] == "even":
        return [i * (n // s) for i in range(s + 1)]
    covered = n - n // 50                                     # the rows behind the last segment are padding
    cuts = (torch.rand(s - 1, generator=gen_cpu) * (covered + 1)).long().clamp_(0, covered)
    for k in range(2, s - 1, 11):                             # a segment in eleven has no row, one has a single row
        cuts[k] = cuts[k - 1]
        cuts[k - 2] = min(int(cuts[k]) + 1, covered)
    return [0] + sorted(cuts.tolist()) + [covered]


def _scan_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    n, s, d, dt = case["rows"], case["segments"], case["width"], _DT[case["dtype"]]
    z = torch.randn(n, 2 * d, generator=gen, device=dev)
    z[:, d:] += torch.linspace(0.0, 6.0, d, device=dev)       # from short memories (a = 0.5) to long ones (a = 0.998)
    z = z.to(dt)
    x, gate = (z[:, :d], z[:, d:]) if case["packed"] else (z[:, :d].contiguous(), z[:, d:].contiguous())
    h0 = torch.randn(s, d, generator=gen, device=dev) * 0.3
    st = {"case": case, "x": x, "gate": gate, "h0": h0}
    if case["op"] == "step":
        return st
    ptr = _segment_rows(case, torch.Generator().manual_seed(seed))
    st["rowptr"] = torch.tensor(ptr, dtype=torch.int32, device=dev)
    st["longest"] = max(b - a for a, b in zip(ptr, ptr[1:]))
    if case["op"] == "scan_train":
        for k in ("x", "gate", "h0"):
            st[k] = st[k].detach().requires_grad_(True)
        st["dh"] = torch.randn(n, d, generator=gen, device=dev).to(dt)
        st["dlast"] = torch.randn(s, d, generator=gen, device=dev)
    return st


def prepare(case, seed):
    return _lookup_inputs(case, seed) if case["op"].startswith("lookup") else _scan_inputs(case, seed)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_lookup(st):
    w, ids, scale = st["weight"].detach(), st["ids"].long(), st["scale"]
    v = w.shape[0]
    there = (ids >= 0) & (ids < v)
    row = torch.where(there, ids, torch.zeros_like(ids))
    out = (w[row].float() * scale * there[:, None]).to(w.dtype)
    if st["case"]["op"] == "lookup":
        return out
    g = st["dout"].float()
    if v <= 32:                                               # few long sums: one masked sum for each
        dw = torch.stack([torch.where((ids == k)[:, None], g, torch.zeros_like(g)).sum(0) for k in range(v)])
    else:
        dw = torch.zeros(v + 1, w.shape[1], device=w.device)
        dw = dw.index_add_(0, torch.where(there, ids, torch.full_like(ids, v)), g)[:v]
    return out, (dw * scale).to(w.dtype)


def _doubling(a, b, longest):
    """h_t = a_t h_{t-1} + b_t down the rows, h before the first row zero: spans of 1, 2, 4, .. rows joined."""
    span = 1
    while span < longest:
        nb, na = b.clone(), a.clone()
        nb[span:] += a[span:] * b[:-span]
        na[span:] *= a[:-span]
        a, b, span = na, nb, 2 * span
    return b


def _plain_scan(st):
    case = st["case"]
    dt = _DT[case["dtype"]]
    x, gate, h0 = st["x"].detach().float(), st["gate"].detach().float(), st["h0"].detach()
    n = x.shape[0]
    ptr = st["rowptr"].long()
    rows = torch.arange(n, device=x.device)
    seg = torch.searchsorted(ptr[1:].contiguous(), rows, right=True)
    inside = (seg < h0.shape[0])[:, None]
    seg = seg.clamp_(max=h0.shape[0] - 1)
    lo, hi = ptr[:-1], ptr[1:]
    first, last = (hi - 1, lo) if case["reverse"] else (lo, hi - 1)        # in the order of the recurrence
    at_first, at_last = (rows == first[seg])[:, None], (rows == last[seg])[:, None]
    has = (hi > lo)[:, None]

    def down(t):
        return t.flip(0) if case["reverse"] else t

    a, c = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    b = torch.where(at_first, a * h0[seg] + c * x, c * x) * inside
    link = torch.where(at_first | ~inside, torch.zeros_like(a), a)
    h = down(_doubling(down(link), down(b), st["longest"]))
    h_last = torch.where(has, h[last.clamp(0, n - 1)], h0)
    if case["op"] == "scan":
        return h.to(dt), h_last
    dh, dlast = st["dh"].float(), st["dlast"]
    g = torch.where(at_last, dh + dlast[seg], dh) * inside
    zero = torch.zeros_like(a[:1])
    nxt = torch.cat([zero, a[:-1]]) if case["reverse"] else torch.cat([a[1:], zero])
    back = torch.where(at_last | ~inside, torch.zeros_like(a), nxt)
    lam = down(_doubling(down(back).flip(0), down(g).flip(0), st["longest"]).flip(0))
    prev = torch.cat([h[1:], zero]) if case["reverse"] else torch.cat([zero, h[:-1]])
    prev = torch.where(at_first, h0[seg], prev)
    dx, dgate = c * lam, lam * (prev - x) * a * c * inside
    dh0 = torch.where(has, (a * lam)[first.clamp(0, n - 1)], dlast)
    return h.to(dt), h_last, dx.to(dt), dgate.to(dt), dh0


def _plain_step(st):
    x, gate = st["x"].float(), st["gate"].float()
    state = st["h0"] / (1 + torch.exp(-gate)) + x / (1 + torch.exp(gate))
    return state.to(st["x"].dtype), state


# ------------------------------------------------------------------------------------------------ the package's operators
def _own_run(st):
    from building_gan_amd import ops
    op = st["case"]["op"]
    if op == "lookup":
        return ops.embedding(st["weight"], st["ids"], st["scale"])
    if op == "lookup_train":
        out = ops.embedding(st["weight"], st["ids"], st["scale"])
        return out, torch.autograd.grad(out, st["weight"], st["dout"])[0]
    if op == "step":
        return ops.gated_scan_step(st["x"], st["gate"], st["h0"])
    h, h_last = ops.gated_scan(st["x"], st["gate"], st["rowptr"], st["h0"], reverse=st["case"]["reverse"])
    if op == "scan":
        return h, h_last
    return (h.detach(), h_last.detach()) + torch.autograd.grad((h, h_last), (st["x"], st["gate"], st["h0"]),
                                                               (st["dh"], st["dlast"]))


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    return _plain_lookup(state) if op.startswith("lookup") else _plain_step(state) if op == "step" else _plain_scan(state)


def work(case):
    b, d = _BYTES[case["dtype"]], case["width"]
    if case["op"].startswith("lookup"):
        n, v = case["tokens"], case["vocab"]
        k = torch.arange(v, dtype=torch.float64)
        p = torch.log((k + 2) / (k + 1)) / math.log(v + 1) if case["skew"] else torch.full_like(k, 1.0 / v)
        touched = float((1 - torch.exp(n * torch.log1p(-p.clamp(max=1 - 1e-12)))).sum())     # table rows that occur
        size = n * (8 if case["ids"] == "i64" else 4) + (touched + n) * d * b
        if case["op"] == "lookup":
            return {"bytes": size, "flops": n * d}
        return {"bytes": size + (n + v) * d * b, "flops": 2 * n * d}
    n, s = case["rows"], case["segments"]
    if case["op"] == "step":
        return {"bytes": n * d * (3 * b + 8), "flops": 12 * n * d}
    if case["op"] == "scan":
        return {"bytes": 3 * n * d * b + 8 * s * d, "flops": 12 * n * d}
    return {"bytes": 8 * n * d * b + 20 * s * d, "flops": 42 * n * d}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0: rows cut into about sqrt(n) pieces, walked row by row side by side, then the
    pieces one after another."""
    n, d = a.shape
    length = max(1, math.isqrt(n))
    pieces = -(-n // length)
    pad = pieces * length - n
    a = torch.cat([a, a.new_ones(pad, d)]).view(pieces, length, d)
    b = torch.cat([b, b.new_zeros(pad, d)]).view(pieces, length, d)
    inner, factor = torch.empty_like(b), torch.empty_like(a)
    h, f = b.new_zeros(pieces, d), a.new_ones(pieces, d)
    for t in range(length):
        h = a[:, t] * h + b[:, t]
        f = f * a[:, t]
        inner[:, t], factor[:, t] = h, f
    carry = b.new_zeros(d)
    for p in range(pieces):
        inner[p] += factor[p] * carry
        carry = inner[p, -1]
    return inner.view(-1, d)[:n]


def _exact_scan(case, seed):
    st = _scan_inputs(case, seed)
    rev = case["reverse"]
    x, gate, h0 = (st[k].detach().double() for k in ("x", "gate", "h0"))
    ptr = st["rowptr"].tolist()
    covered = ptr[-1]
    if rev:                                                   # the same recurrence on the rows in the opposite order
        ptr_f = [covered - p for p in reversed(ptr)]
        x, gate, h0 = x[:covered].flip(0), gate[:covered].flip(0), h0.flip(0)
    else:
        ptr_f, x, gate = ptr, x[:covered], gate[:covered]
    some = [s for s in range(len(ptr_f) - 1) if ptr_f[s + 1] > ptr_f[s]]
    idx = torch.tensor(some, device=x.device)
    heads = torch.tensor([ptr_f[s] for s in some], device=x.device)
    tails = torch.tensor([ptr_f[s + 1] - 1 for s in some], device=x.device)
    a, c = torch.sigmoid(gate), torch.sigmoid(-gate)
    b = c * x
    b[heads] += a[heads] * h0[idx]
    link = a.clone()
    link[heads] = 0.0
    h = _exact_recurrence(link, b)
    last = h0.clone()
    last[idx] = h[tails]

    def rows(t):                                              # back to the order and number of the rows
        t = t.flip(0) if rev else t
        return torch.cat([t, t.new_zeros(case["rows"] - covered, t.shape[1])])

    def segs(t):
        return t.flip(0) if rev else t

    if case["op"] == "scan":
        return rows(h), segs(last)
    dh, dlast = st["dh"].double()[:covered], st["dlast"].double()
    if rev:
        dh, dlast = dh.flip(0), dlast.flip(0)
    g = dh.clone()
    g[tails] += dlast[idx]
    coupling = torch.zeros_like(a)
    coupling[:-1] = a[1:]
    coupling[tails] = 0.0
    lam = _exact_recurrence(coupling.flip(0), g.flip(0)).flip(0)
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[heads] = h0[idx]
    dh0 = dlast.clone()
    dh0[idx] = a[heads] * lam[heads]
    return rows(h), segs(last), rows(c * lam), rows(lam * (before - x) * a * c), segs(dh0)


def exact(case, seed):
    if case["op"] == "step":
        st = _scan_inputs(case, seed)
        x, gate, state = st["x"].double(), st["gate"].double(), st["h0"].double()
        state = torch.sigmoid(gate) * state + torch.sigmoid(-gate) * x
        return state, state
    if not case["op"].startswith("lookup"):
        return _exact_scan(case, seed)
    st = _lookup_inputs(case, seed)
    w, ids = st["weight"].detach(), st["ids"].long()
    out = torch.zeros(ids.shape[0], w.shape[1], dtype=torch.float64, device=w.device)
    keep = torch.nonzero((ids >= 0) & (ids < w.shape[0]))[:, 0]
    out[keep] = w[ids[keep]].double() * st["scale"]
    if case["op"] == "lookup":
        return out
    order = torch.sort(ids[keep], stable=True)
    g = st["dout"].double()[keep[order.indices]]
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    found, counts = torch.unique_consecutive(order.values, return_counts=True)
    end = torch.cumsum(counts, 0)
    start = end - counts
    total, at = [], 0
    step = max(1, (1 << 24) // w.shape[1])                    # running sums over bounded numbers of rows
    sums = torch.zeros(found.shape[0], w.shape[1], dtype=torch.float64, device=w.device)
    while at < g.shape[0]:
        stop = min(g.shape[0], at + step)
        run_sum = torch.cat([g.new_zeros(1, g.shape[1]), torch.cumsum(g[at:stop], 0)])
        sums += run_sum[end.clamp(at, stop) - at] - run_sum[start.clamp(at, stop) - at]
        at = stop
    dw[found] = sums * st["scale"]
    return out, dw
