"""Table lookup (ops.embedding) and gated scan (ops.gated_scan, ops.gated_scan_step) against plain float64 loops.

Tolerances.  u = 2^-24 is half a step of fp32, ``half(t)`` half a step of the element type; results are fp32 values rounded
to the type once.
 * lookup: one product and one rounding of the scale to fp32 (2 u) and the rounding to the type.
 * lookup gradient: m terms added in fp32 in some order: m u sum|g|, then the scale (2 u) and the rounding.
 * a = sigmoid(g) and c = sigmoid(-g): with e = exp(-|g|) the smaller one is e / (1 + e), from exp2 and a reciprocal (1 ulp = 2 u
   each) with a compensated argument: e within 4 u, of which e / (1 + e) takes half to all, then a sum, a reciprocal and a
   product: within 8 u (6 u where both are 1/2).  The larger one is 1 minus it: within 7 u.  (Below the smallest normal number,
   behind |g| = 87.3, the smaller one is 0.)  One step of the recurrence adds at most 12 u of a |h| + c |x| (8 u and two
   roundings), and what a step has wrong decays with the a's behind it: ``err_t = a_t err_{t-1} + 12 u (a |h| + c |x|)``.
   Joining row groups, waves, 8 tiles to a group, 8 groups to a block and block to block (at most 24 + tiles / 64 joins of
   tiles of 128 rows and more, factors at most 1; the bound takes 64 + rows / (32 * 128)) adds 2 u max|h| each.
 * the backward recurrence alike, with the sums of |terms| in the place of |h|; dx and dgate multiply a few factors each
   known to the errors above.
"""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half(t):
    return torch.finfo(t).eps / 2


def floor_of(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps      # a rounding among the subnormal numbers


def within(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), "%s: %d of %d beyond the bound, worst %.3g times it" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp_min(1e-300)).max()))


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_operands_on_the_cpu_are_refused():
    from building_gan_amd import _lib, ops
    w, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.embedding(w, ids), lambda: ops.embedding_grad_raw(torch.zeros(3, 8), ids, 4),
                 lambda: ops.gated_scan(w, w), lambda: ops.gated_scan_step(w, w, w),
                 lambda: ops.embedding(w.clone().requires_grad_(True), ids),
                 lambda: ops.gated_scan(w.clone().requires_grad_(True), w)):
        with pytest.raises(_lib.BganError):
            call()
    with pytest.raises(IndexError):
        ops.embedding(w, ids + 4, validate=True)
    with pytest.raises(IndexError):
        ops.embedding(w, ids - 1, validate=True)


def test_entry_points_refuse_bad_arguments_before_any_launch():
    """Status codes of the C entry points for what they do not take (no kernel is launched, so no GPU is needed)."""
    from building_gan_amd import _lib
    lib = _lib.load()
    p = 1 << 20                                              # an address that is never read
    fwd = lambda **k: lib.bg_embedding_fwd(*{**dict(dt=0, w=p, ldw=8, V=4, ids=p, i64=1, n=3, D=8, scale=1.0, out=p, ldo=8, s=None), **k}.values())
    assert fwd(dt=3) == -1 and fwd(ldw=7) == -1 and fwd(ldo=7) == -1 and fwd(n=-1) == -1 and fwd(w=None) == -1
    assert fwd(ids=None) == -1 and fwd(out=None) == -1 and fwd(V=-1) == -1
    assert fwd(D=1 << 16, ldw=1 << 16, ldo=1 << 16) == -2 and fwd(n=1 << 40) == -2
    assert fwd(n=0) == 0 and fwd(D=0, ldw=0, ldo=0) == 0
    size = lib.bg_embedding_bwd_workspace(0, 3, 4, 8)
    assert size > 0 and lib.bg_embedding_bwd_workspace(0, 0, 4, 8) == 0
    bwd = lambda **k: lib.bg_embedding_bwd(*{**dict(dt=0, g=p, ldg=8, ids=p, i64=1, n=3, D=8, V=4, scale=1.0, dw=p, ws=p, size=size, s=None), **k}.values())
    assert bwd(dt=-1) == -1 and bwd(ldg=7) == -1 and bwd(dw=None) == -1 and bwd(ws=None) == -1 and bwd(g=None) == -1
    assert bwd(dw=p + 4) == -3 and bwd(ws=p + 8) == -3 and bwd(size=size - 1) == -5
    assert bwd(V=(1 << 31) - 1) == -2 and bwd(n=(1 << 30) + 1) == -2 and bwd(D=1 << 16, ldg=1 << 16) == -2
    assert bwd(V=0) == 0 and bwd(D=0, ldg=0) == 0
    size = lib.bg_gated_scan_workspace(10, 8)
    heads = lib.bg_gated_scan_heads(10, 8)
    assert size > 0 and heads >= 2 * 8 and lib.bg_gated_scan_workspace(0, 8) == 0
    scan = lambda **k: lib.bg_gated_scan_fwd(*{**dict(dt=0, x=p, ldx=8, g=p, ldg=8, rp=p, S=2, N=10, D=8, h0=None, rev=0, h=p, ldh=8, hl=p,
                                                      heads=None, ws=p, size=size, s=None), **k}.values())
    assert scan(dt=7) == -1 and scan(ldx=7) == -1 and scan(ldg=7) == -1 and scan(ldh=7) == -1 and scan(x=None) == -1
    assert scan(ws=None) == -1 and scan(ws=p + 8) == -3 and scan(size=size - 1) == -5 and scan(S=-1) == -1
    assert scan(rp=None, S=3) == -1 and scan(rp=None, S=0) == -1 and scan(N=1 << 31) == -2 and scan(D=1 << 21, ldx=1 << 21, ldg=1 << 21, ldh=1 << 21) == -2
    assert scan(D=0, ldx=0, ldg=0, ldh=0) == 0 and scan(N=0, hl=None) == 0
    back = lambda **k: lib.bg_gated_scan_bwd(*{**dict(dt=0, x=p, ldx=8, g=p, ldg=8, dh=p, lddh=8, dl=None, rp=p, S=2, N=10, D=8, h0=None,
                                                      rev=0, heads=p, dx=p, lddx=8, dg=p, lddg=8, dh0=None, ws=p, size=size, s=None), **k}.values())
    assert back(lddh=7) == -1 and back(lddx=7) == -1 and back(lddg=7) == -1 and back(heads=None) == -1 and back(dx=None) == -1
    assert back(size=size - 1) == -5 and back(ws=p + 4) == -3 and back(dt=5) == -1
    step = lambda **k: lib.bg_gated_scan_step(*{**dict(dt=0, x=p, ldx=8, g=p, ldg=8, st=p, lds=8, n=3, D=8, h=p, ldh=8, so=p, ldso=8, s=None), **k}.values())
    assert step(st=None) == -1 and step(lds=7) == -1 and step(ldso=7) == -1 and step(n=-1) == -1 and step(n=1 << 30) == -2 and step(n=0) == 0


@pytest.mark.gpu
def test_wrappers_refuse_what_does_not_fit(cuda):
    from building_gan_amd import _lib, ops
    w = torch.zeros(4, 8, device=cuda)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda)
    rp = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda)
    bad = [lambda: ops.embedding(w.double(), ids), lambda: ops.embedding(w[0], ids), lambda: ops.embedding(w, ids.float()),
           lambda: ops.embedding(w, ids.cpu()), lambda: ops.embedding_grad_raw(torch.zeros(4, 8, device=cuda), ids, 4),
           lambda: ops.embedding_grad_raw(torch.zeros(3, 8, device=cuda), ids, -1),
           lambda: ops.gated_scan(w, w.half()), lambda: ops.gated_scan(w, w[:3]), lambda: ops.gated_scan(w, w, rp.long()),
           lambda: ops.gated_scan(w, w, rp.cpu()), lambda: ops.gated_scan(w, w, rp, h0=torch.zeros(3, 8, device=cuda)),
           lambda: ops.gated_scan(w, w, rp, h0=torch.zeros(2, 8, device=cuda, dtype=torch.float16)),
           lambda: ops.gated_scan(w.view(2, 2, 8), w.view(2, 2, 8), rp), lambda: ops.gated_scan(w[0], w[0]),
           lambda: ops.gated_scan_step(w, w, w.half()), lambda: ops.gated_scan_step(w, w, w[:3]),
           lambda: ops.gated_scan_step(w, w, w, state_out=w[:3]),
           lambda: ops.gated_scan_raw(w, w, 3)]
    for k, call in enumerate(bad):
        with pytest.raises(_lib.BganError):
            call()
            pytest.fail("call %d was accepted" % k)
    buf = torch.zeros(5, 8, device=cuda)
    with pytest.raises(_lib.BganError):
        ops.gated_scan_step(w, w, buf[:4], state_out=buf[1:])
    with pytest.raises(IndexError):
        ops.embedding(w, ids + 4, validate=True)
    assert torch.equal(ops.embedding(w, ids + 3, validate=True), w[ids + 3])


# ------------------------------------------------------------------------------------------------ lookup
def lookup_case(V, D, n, dtype, seed, kind="uniform", ids_dtype=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=gen).to(dtype)
    g = torch.randn(n, D, generator=gen).to(dtype)
    ids = torch.randint(0, V, (n,), generator=gen)
    if kind == "one":
        ids[:] = V - 1
    elif kind == "hot":                                     # three tokens in four are the same one
        ids[torch.rand(n, generator=gen) < 0.75] = V // 2
    elif kind == "missing":
        ids[::3] = torch.tensor([-1, V, -(2 ** 31), 2 ** 31 - 1])[torch.arange(len(ids[::3])) % 4]
    elif kind == "none":
        ids[:] = -1
    return w, ids.to(ids_dtype), g


def check_lookup(cuda, w, ids, g, scale):
    from building_gan_amd import ops
    V, D = w.shape
    dt = w.dtype
    wd = w.to(cuda).requires_grad_(True)
    out = ops.embedding(wd, ids.to(cuda), scale)
    (dw,) = torch.autograd.grad(out, wd, g.to(cuda))
    assert out.dtype == dt and dw.dtype == dt and out.shape == (*ids.shape, D)
    i = ids.long().reshape(-1)
    there = (i >= 0) & (i < V)
    want = torch.zeros(i.numel(), D, dtype=torch.float64)
    want[there] = w.double()[i[there]] * scale
    within(out.reshape(-1, D), want, want.abs() * (half(dt) + 2.1 * U) + floor_of(dt), "lookup")
    gd = g.reshape(-1, D).double()[there]
    s = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i[there], gd)
    sa = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i[there], gd.abs())
    m = torch.zeros(V, 1, dtype=torch.float64).index_add_(0, i[there], torch.ones(len(gd), 1, dtype=torch.float64))
    within(dw, s * scale, (s.abs() * half(dt) + sa * (m + 2.1) * U * 1.01) * scale + floor_of(dt), "lookup gradient")
    assert not dw.detach().cpu()[(m == 0)[:, 0]].any(), "a row without tokens has a gradient"
    with torch.no_grad():
        assert torch.equal(ops.embedding(wd, ids.to(cuda), scale), out)
    assert torch.equal(ops.embedding_grad_raw(g.to(cuda), ids.to(cuda), V, scale), dw), "not reproducible"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,D,n,kind", [
    (7, 128, 1440, "uniform"), (20, 128, 333, "uniform"), (7, 4, 5000, "hot"), (1, 64, 257, "uniform"), (1000, 32, 1, "uniform"),
    (1000, 520, 700, "missing"), (513, 33, 1500, "missing"), (300, 1, 2000, "hot"), (2, 7, 9, "none"), (40000, 16, 5000, "hot"),
    (300000, 8, 3000, "uniform"), (511, 72, 1024, "one"), (512, 8, 1025, "one"), (5000, 256, 2049, "uniform")])
def test_lookup_and_gradient_match_float64(cuda, V, D, n, kind, dtype):
    w, ids, g = lookup_case(V, D, n, dtype, V + D + n, kind, torch.int32 if n % 2 else torch.int64)
    check_lookup(cuda, w, ids, g, 0.75 if D % 2 else 11.313708498984761)


@pytest.mark.gpu
@pytest.mark.parametrize("V,D,n,kind", [(70000, 8, 70001, "hot"), (70000, 12, 300000, "uniform"), (6, 24, 200000, "uniform"),
                                        (31, 16, 70000, "hot"), (100, 40, 131072, "one")])
def test_lookup_gradient_with_many_tokens(cuda, V, D, n, kind):
    """More tokens than one scan of the tile counts covers, runs over many tiles."""
    w, ids, g = lookup_case(V, D, n, torch.float32, n, kind)
    check_lookup(cuda, w, ids, g, 1.0)


@pytest.mark.gpu
def test_lookup_strides_shapes_and_empty_operands(cuda):
    from building_gan_amd import ops
    gen = torch.Generator().manual_seed(3)
    big = torch.randn(50, 40, generator=gen).to(cuda)
    ids = torch.randint(0, 50, (4, 5, 6), generator=gen).to(cuda)
    for w in (big[:, :24], big[:, 3:27], big[::2, :24], big.t()[:40]):      # pitched, unaligned, strided rows, transposed
        i = ids % w.shape[0]
        assert torch.equal(ops.embedding(w, i), w[i])
        assert torch.equal(ops.embedding(w, i.transpose(0, 2)), w[i.transpose(0, 2)])
    w = big.clone().requires_grad_(True)
    ops.embedding(w, ids, 2.0).sum().backward()                              # a gradient without strides of its own
    assert torch.equal(w.grad[:, 0].cpu(), 2.0 * torch.bincount(ids.flatten().cpu(), minlength=50).float())
    gbig = torch.randn(120, 60, generator=gen).to(cuda)
    flat = ids.flatten()
    for gg in (gbig[:, 1:41], gbig[:, :40]):                                 # a pitch, with and without alignment
        assert torch.equal(ops.embedding_grad_raw(gg, flat, 50), ops.embedding_grad_raw(gg.contiguous(), flat, 50))
    assert ops.embedding(big, ids[:0]).shape == (0, 5, 6, 40)
    assert ops.embedding(big[:, :0], ids).shape == (4, 5, 6, 0)
    assert not ops.embedding_grad_raw(gbig[:0, :40], flat[:0], 50).any()
    assert ops.embedding_grad_raw(gbig[:, :40], flat, 0).shape == (0, 40)
    assert not ops.embedding(big[:0], ids).any()


@pytest.mark.gpu
def test_lookup_not_finite_values_stay_where_they_are(cuda):
    from building_gan_amd import ops
    w = torch.ones(6, 16, device=cuda)
    w[2], w[3] = float("nan"), float("inf")
    ids = torch.tensor([0, 2, -1, 3, 99, 5], device=cuda)
    out = ops.embedding(w, ids)
    assert torch.equal(out[[0, 5]], w[[0, 5]]) and out[1].isnan().all() and out[3].isinf().all() and not out[[2, 4]].any()
    g = torch.ones(6, 16, device=cuda)
    g[2] = g[4] = float("nan")                                               # behind the missing tokens
    g[1] = float("inf")
    dw = ops.embedding_grad_raw(g, ids, 6)
    assert torch.equal(dw.sum(1).cpu(), torch.tensor([16.0, 0, float("inf"), 16, 0, 16]))


@pytest.mark.gpu
def test_lookup_twice_differentiable(cuda):
    """The gradient's own backward is the lookup (both are linear)."""
    from building_gan_amd import ops
    w = torch.randn(9, 12, device=cuda, requires_grad=True)
    ids = torch.randint(0, 9, (40,), device=cuda)
    v = torch.randn(40, 12, device=cuda, requires_grad=True)
    (dw,) = torch.autograd.grad(ops.embedding(w, ids, 3.0), w, v, create_graph=True)
    t = torch.randn(9, 12, device=cuda)
    (dv,) = torch.autograd.grad(dw, v, t)
    assert torch.equal(dv, 3.0 * t[ids])


# ------------------------------------------------------------------------------------------------ scan
def scan_reference(x, gate, ptr, h0, reverse, dh, dlast):
    """float64 loops: values and error bounds (before the rounding to the type) of h, h_last, dx, dgate, dh0."""
    N, D = x.shape
    S = len(ptr) - 1
    x, gate = x.double(), gate.double()
    a, c = torch.sigmoid(gate), torch.sigmoid(-gate)
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)
    h0 = z(S, D) if h0 is None else h0.double()
    dlast = z(S, D) if dlast is None else dlast.double()
    dh = z(N, D) if dh is None else dh.double()
    h, e, hp, ep, lam, el, big = z(N, D), z(N, D), z(N, D), z(N, D), z(N, D), z(N, D), z(N, D)
    hl, ehl, d0, ed0 = h0.clone(), z(S, D), dlast.clone(), z(S, D)
    top = max([float(t.abs().max()) for t in (x, h0) if t.numel()] + [0.0])
    joins = 64 + N / (32 * 128)
    for s in range(S):
        rows = list(range(ptr[s], ptr[s + 1]))
        if reverse:
            rows.reverse()
        st, er = h0[s], z(D)
        for t in rows:
            hp[t], ep[t] = st, er
            er = a[t] * er + 12 * U * (a[t] * st.abs() + c[t] * x[t].abs())
            st = a[t] * st + c[t] * x[t]
            h[t], e[t] = st, er
        hl[s], ehl[s] = st, er
        mu, em, sz = dlast[s], z(D), dlast[s].abs()
        for t in reversed(rows):
            lam[t] = dh[t] + mu
            big[t] = dh[t].abs() + sz
            el[t] = em + U * big[t]
            mu, sz, em = a[t] * lam[t], a[t] * big[t], a[t] * el[t] + 12 * U * a[t] * big[t]
        d0[s], ed0[s] = mu, em
    jh = 2 * U * joins * top
    jl = 2 * U * joins * (float(big.max()) if N else 0.0)
    e, ep, ehl = e + jh, ep + jh, ehl + jh
    el, ed0 = el + jl, ed0 + jl
    ac = a * c
    dx, dg = c * lam, lam * (hp - x) * ac
    edx = c * el + 12 * U * c * big
    edg = ac * (el * (hp - x).abs() + big * (ep + U * (hp.abs() + x.abs())) + 25 * U * big * (hp - x).abs() + el * ep)
    return (h, hl, dx, dg, d0), (e, ehl, edx, edg, ed0)


def scan_case(N, D, ptr, dtype, seed, h0=True, slow=False):
    gen = torch.Generator().manual_seed(seed)
    z = torch.randn(N, 2 * D, generator=gen)
    z[:, D:] += torch.linspace(-2.0, 9.0 if slow else 5.0, D)
    z = z.to(dtype)
    S = len(ptr) - 1
    return dict(z=z, x=z[:, :D], gate=z[:, D:], h0=torch.randn(S, D, generator=gen) if h0 else None,
                dh=torch.randn(N, D, generator=gen).to(dtype), dlast=torch.randn(S, D, generator=gen))


def check_scan(cuda, c, ptr, reverse=False, use_dh=True, use_dlast=True, packed=True, rowptr="ptr"):
    from building_gan_amd import ops
    dt = c["x"].dtype
    z = c["z"].to(cuda)
    D = c["x"].shape[1]
    x, gate = (z[:, :D], z[:, D:]) if packed else (z[:, :D].contiguous(), z[:, D:].contiguous())
    x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    h0 = None if c["h0"] is None else c["h0"].to(cuda).requires_grad_(True)
    rp = torch.tensor(ptr, dtype=torch.int32, device=cuda) if rowptr == "ptr" else rowptr
    dh, dlast = c["dh"] if use_dh else None, c["dlast"] if use_dlast else None
    h, hl = ops.gated_scan(x, gate, rp, h0, reverse)
    outs, grads = [], []
    if use_dh:
        outs.append(h), grads.append(dh.to(cuda))
    if use_dlast:
        outs.append(hl), grads.append(dlast.to(cuda))
    got = torch.autograd.grad(outs, [x, gate] + ([] if h0 is None else [h0]), grads)
    want, err = scan_reference(c["x"], c["gate"], ptr, c["h0"], reverse, dh, dlast)
    for name, g, w, e, t in zip(("h", "h_last", "dx", "dgate", "dh0"), (h, hl) + got, want, err, (dt, torch.float32, dt, dt, torch.float32)):
        assert g.dtype == t
        within(g, w, e * 1.01 + w.abs() * half(t) + floor_of(t), name)
    with torch.no_grad():                                    # without heads, and again: the same bits
        h2, hl2 = ops.gated_scan(x, gate, rp, h0, reverse)
    assert torch.equal(h2, h) and torch.equal(hl2, hl)
    return (h, hl) + got


RAGGED = [0, 0, 1, 40, 40, 40, 41, 200, 201, 460, 460]       # no rows, one row, first and last segment empty


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("D", [1, 3, 8, 33, 64, 100, 128, 260])
def test_scan_and_gradients_match_float64(cuda, D, reverse, dtype):
    c = scan_case(460, D, RAGGED, dtype, D)
    check_scan(cuda, c, RAGGED, reverse, packed=D % 8 != 0)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("N,D,ptr", [(300, 36, [5, 5, 100, 260]), (300, 8, [300, 300]), (17, 5, [0, 17]), (1, 4, [0, 1]),
                                     (2, 130, [0, 1, 2]), (128, 128, [0, 128]), (129, 132, [0, 128, 129]), (700, 68, [0, 0, 700, 700]),
                                     (1030, 12, [0, 512, 1030]), (9000, 8, [0, 100, 8900]), (5000, 132, [0, 5000])])
def test_scan_rows_behind_the_segments_and_tile_edges(cuda, N, D, ptr, reverse):
    c = scan_case(N, D, ptr, torch.float32, N + D, slow=True)
    got = check_scan(cuda, c, ptr, reverse)
    for t in (got[0], got[2], got[3]):
        assert not t[:ptr[0]].any() and not t[ptr[-1]:].any(), "a row in no segment is not zero"


@pytest.mark.gpu
@pytest.mark.parametrize("h0,use_dh,use_dlast", [(False, True, True), (True, False, True), (True, True, False), (False, False, True)])
def test_scan_without_optional_operands(cuda, h0, use_dh, use_dlast):
    c = scan_case(460, 20, RAGGED, torch.float32, 5, h0=h0)
    check_scan(cuda, c, RAGGED, use_dh=use_dh, use_dlast=use_dlast)


# Values only, and the comparison for B == 1 never runs: test_scan_of_a_batch_and_its_gradients has both.
@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_equal_segments_and_batches(cuda, reverse):
    from building_gan_amd import ops
    B, T, D = 6, 77, 24
    c = scan_case(B * T, D, list(range(0, B * T + 1, T)), torch.float32, 11)
    ptr = list(range(0, B * T + 1, T))
    a = check_scan(cuda, c, ptr, reverse)
    b = check_scan(cuda, c, ptr, reverse, rowptr=None) if B == 1 else None
    x, gate, h0 = c["x"].to(cuda), c["gate"].to(cuda), c["h0"].to(cuda)
    h, hl = ops.gated_scan(x.view(B, T, D), gate.view(B, T, D), h0=h0, reverse=reverse)
    assert torch.equal(h.view(-1, D), a[0]) and torch.equal(hl, a[1]) and b is None
    z = c["z"].to(cuda).view(B, T, 2 * D)
    h, hl = ops.gated_scan(z[..., :D], z[..., D:], h0=h0, reverse=reverse)
    assert torch.equal(h.view(-1, D), a[0])
    h, hl = ops.gated_scan(x.view(B, T, D).transpose(0, 1), gate.view(B, T, D).transpose(0, 1), reverse=reverse)   # copied first
    e, el = ops.gated_scan(x.view(B, T, D).transpose(0, 1).contiguous(), gate.view(B, T, D).transpose(0, 1).contiguous(), reverse=reverse)
    assert torch.equal(h, e) and torch.equal(hl, el)
    one, onel = ops.gated_scan(x, gate, reverse=reverse)     # no row pointer: one segment
    two, twol = ops.gated_scan(x, gate, torch.tensor([0, B * T], dtype=torch.int32, device=cuda), reverse=reverse)
    assert torch.equal(one, two) and torch.equal(onel, twol)


@pytest.mark.gpu
def test_scan_of_nothing(cuda):
    from building_gan_amd import ops
    h0 = torch.randn(3, 8, device=cuda, requires_grad=True)
    x = torch.zeros(0, 8, device=cuda, requires_grad=True)
    h, hl = ops.gated_scan(x, x.detach(), torch.zeros(4, dtype=torch.int32, device=cuda), h0)
    assert h.shape == (0, 8) and torch.equal(hl, h0)
    g = torch.randn(3, 8, device=cuda)
    assert torch.equal(torch.autograd.grad(hl, h0, g)[0], g)
    h, hl = ops.gated_scan(x.detach(), x.detach())
    assert h.shape == (0, 8) and hl.shape == (1, 8) and not hl.any()
    e = torch.zeros(3, 0, 8, device=cuda)
    h, hl = ops.gated_scan(e, e, h0=h0.detach())
    assert h.shape == (3, 0, 8) and torch.equal(hl, h0)
    w = torch.zeros(5, 0, device=cuda)
    assert ops.gated_scan(w, w)[0].shape == (5, 0)
    y = torch.ones(5, 8, device=cuda)                        # rows, but no segment
    h, hl = ops.gated_scan(y, y, torch.zeros(1, dtype=torch.int32, device=cuda))
    assert not h.any() and hl.shape == (0, 8)


# (What takes two rounds is the marking of a tile's borders, a lane for each segment; its first segment is found by bisection.)
@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_with_many_segments(cuda, reverse):
    """More segments than a workgroup has threads: the search for a tile's first segment takes two rounds."""
    gen = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 3, (3000,), generator=gen)
    ptr = [0] + torch.cumsum(lens, 0).tolist()
    c = scan_case(ptr[-1], 8, ptr, torch.float32, 2)
    check_scan(cuda, c, ptr, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_not_finite_values_stay_in_their_segment_and_column(cuda, reverse):
    from building_gan_amd import ops
    ptr = [0, 150, 151, 400, 600]
    c = scan_case(620, 12, ptr, torch.float32, 4)
    x, gate, h0 = c["x"].clone(), c["gate"].clone(), c["h0"].clone()
    clean = [t.clone() for t in ops.gated_scan(x.to(cuda), gate.to(cuda), torch.tensor(ptr, dtype=torch.int32, device=cuda), h0.to(cuda), reverse)]
    x[160, 3] = float("nan")
    x[605, 4] = gate[610, 5] = float("nan")                  # rows in no segment
    h0[0, 7] = float("inf")
    rp = torch.tensor(ptr, dtype=torch.int32, device=cuda)
    xs, gs, hs = x.to(cuda).requires_grad_(True), gate.to(cuda).requires_grad_(True), h0.to(cuda).requires_grad_(True)
    h, hl = ops.gated_scan(xs, gs, rp, hs, reverse)
    dx, dg, d0 = torch.autograd.grad((h, hl), (xs, gs, hs), (torch.ones_like(h), torch.ones_like(hl)))
    touched = torch.zeros(620, 12, dtype=torch.bool)
    touched[151:400, 3] = True
    touched[0:150, 7] = True
    same = (h == clean[0]).cpu()
    assert same[~touched].all() and not h[600:].any() and not dx[600:].any() and not dg[600:].any()
    assert h[160 if reverse else 399, 3].isnan() and hl[2, 3].isnan()
    assert torch.isfinite(dx).all() and torch.isfinite(d0).all() and torch.isfinite(dg.cpu()[~touched]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_scan_saturated_gates(cuda, dtype):
    """Gates that hold the state (a = 1 exactly, c = 0) and that replace it (a = 0)."""
    from building_gan_amd import ops
    inf = float("inf")
    x = torch.arange(1.0, 7.0, device=cuda).view(6, 1).expand(6, 8).contiguous().to(dtype)
    gate = torch.tensor([-inf, inf, 200.0, -200.0, inf, -inf], device=cuda).view(6, 1).expand(6, 8).contiguous().to(dtype)
    x.requires_grad_(True), gate.requires_grad_(True)
    h, hl = ops.gated_scan(x, gate)
    assert h[:, 0].tolist() == [1, 1, 1, 4, 4, 6] and hl[0, 0] == 6
    dx, dg = torch.autograd.grad(h, (x, gate), torch.ones_like(h))
    assert dx[:, 0].tolist() == [3, 0, 0, 2, 0, 1] and not dg.any()
    gate = torch.tensor([30.0, -30.0, 80.0, -80.0, 1e-30, -1e-30], device=cuda).view(6, 1).contiguous()
    one = torch.ones(6, 1, device=cuda)
    c1 = ops.gated_scan_step(one, gate, torch.zeros(6, 1, device=cuda))[1].cpu().double()      # sigmoid(-gate) itself
    a1 = ops.gated_scan_step(torch.zeros_like(one), gate, one)[1].cpu().double()
    g = gate.cpu().double()
    within(c1, torch.sigmoid(-g), torch.sigmoid(-g) * 12 * U, "sigmoid(-gate)")
    within(a1, torch.sigmoid(g), torch.sigmoid(g) * 12 * U, "sigmoid(gate)")


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_gradients_against_differences(cuda, reverse):
    """<gradient, direction> against central differences of the float64 loops (step 1e-4: their own error is below 1e-7 of
    the derivative's scale)."""
    from building_gan_amd import ops
    ptr = [0, 30, 30, 95, 131]
    c = scan_case(140, 6, ptr, torch.float32, 8)
    x, gate, h0 = (c[k].to(cuda).contiguous().requires_grad_(True) for k in ("x", "gate", "h0"))
    h, hl = ops.gated_scan(x, gate, torch.tensor(ptr, dtype=torch.int32, device=cuda), h0, reverse)
    grads = torch.autograd.grad((h, hl), (x, gate, h0), (c["dh"].to(cuda), c["dlast"].to(cuda)))
    _, err = scan_reference(c["x"], c["gate"], ptr, c["h0"], reverse, c["dh"], c["dlast"])

    def loss(xx, gg, hh):
        v, _ = scan_reference(xx, gg, ptr, hh, reverse, None, None)
        return float((v[0] * c["dh"].double()).sum() + (v[1] * c["dlast"].double()).sum())

    at = [c["x"].double(), c["gate"].double(), c["h0"].double()]
    gen = torch.Generator().manual_seed(1)
    for k in range(3):
        d = torch.randn(at[k].shape, generator=gen, dtype=torch.float64)
        up, dn = list(at), list(at)
        up[k], dn[k] = at[k] + 1e-4 * d, at[k] - 1e-4 * d
        diff = (loss(*up) - loss(*dn)) / 2e-4
        g = grads[k].cpu().double()
        tol = float(((err[2 + k] + g.abs() * U) * d.abs()).sum()) + 1e-7 * float((g * d).abs().sum())
        assert abs(float((g * d).sum()) - diff) <= tol, (k, float((g * d).sum()), diff, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D", [(1, 1), (3, 7), (50, 256), (5, 1028), (9, 2051)])
def test_step_matches_float64_and_the_scan(cuda, n, D, dtype):
    from building_gan_amd import ops
    c = scan_case(n, D, list(range(n + 1)), dtype, n * D)
    z, state = c["z"].to(cuda), c["h0"].to(cuda)
    h, new = ops.gated_scan_step(z[:, :D], z[:, D:], state)
    want, err = scan_reference(c["x"], c["gate"], list(range(n + 1)), c["h0"], False, None, None)
    within(new, want[1], err[1], "state")
    within(h, want[0], err[0] + want[0].abs() * half(dtype) + floor_of(dtype), "h")
    hs, hl = ops.gated_scan(z[:, :D], z[:, D:], torch.arange(n + 1, dtype=torch.int32, device=cuda), state)
    assert torch.equal(hs, h) and torch.equal(hl, new), "a scan over segments of one row is the step"
    kept = state.clone()
    h2, out = ops.gated_scan_step(z[:, :D], z[:, D:], kept, state_out=kept)
    assert out is kept and torch.equal(kept, new) and torch.equal(h2, h)


@pytest.mark.gpu
def test_step_leaves_other_rows_alone(cuda):
    from building_gan_amd import ops
    buf = torch.randn(9, 40, device=cuda)
    before = buf.clone()
    x = torch.randn(4, 36, device=cuda)
    view = buf[2:6, 2:38]                                    # a pitch and no 16-byte alignment
    h, _ = ops.gated_scan_step(x, x, view, state_out=view)
    want = ops.gated_scan_step(x, x, before[2:6, 2:38].contiguous())[1]
    assert torch.equal(view, want)
    buf[2:6, 2:38] = before[2:6, 2:38]
    assert torch.equal(buf, before)
    assert ops.gated_scan_step(x[:0], x[:0], view[:0])[0].shape == (0, 36)


# ------------------------------------------------------------------------------------------------ together
def run_together(dev, seed=0):
    from building_gan_amd.synthetic import make_batch
    from building_gan_amd.plan import build_plan
    g = make_batch("small", seed=seed, ragged=True).to(dev)
    return build_plan(g)


@pytest.mark.gpu
def test_levels_looked_up_scanned_along_stories_and_pooled(cuda):
    """A batch's floor levels -> learned vectors -> state along each graph's voxels -> graph pooling, with gradients, against
    float64 autograd over the same steps."""
    from building_gan_amd import ops
    p = run_together(cuda)
    seg = p.graph_seg if hasattr(p, "graph_seg") else p.story_seg
    N, D = seg.n_cols, 32
    level = p.level
    gen = torch.Generator().manual_seed(2)
    table = (torch.randn(20, 2 * D, generator=gen) * 0.5)
    start = torch.randn(seg.n_rows, D, generator=gen)
    wt, st = table.to(cuda).requires_grad_(True), start.to(cuda).requires_grad_(True)
    z = ops.embedding(wt, level, 1.5)
    h, hl = ops.gated_scan(z[:, :D], z[:, D:], seg.rowptr, st)
    pooled, _ = ops.SegMax.apply(h, seg)
    cot = torch.randn(seg.n_rows, D, generator=gen)
    loss = (pooled * cot.to(cuda)).sum() + (hl * cot.to(cuda)).sum()
    dw, ds = torch.autograd.grad(loss, (wt, st))
    w64, s64 = table.double().requires_grad_(True), start.double().requires_grad_(True)
    z64 = 1.5 * w64[level.cpu().long()]
    ptr = seg.rowptr.tolist()
    best, last = [], []
    for s in range(seg.n_rows):
        state, hs = s64[s], []
        for t in range(ptr[s], ptr[s + 1]):
            a = torch.sigmoid(z64[t, D:])
            state = a * state + (1 - a) * z64[t, :D]
            hs.append(state)
        best.append(torch.stack(hs).max(0).values), last.append(state)
    want = (torch.stack(best) * cot.double()).sum() + (torch.stack(last) * cot.double()).sum()
    dw64, ds64 = torch.autograd.grad(want, (w64, s64))
    # the sums of some hundred products of fp32 factors each known to about 100 u (module docstring: a state's error after many rows)
    torch.testing.assert_close(loss.detach().cpu().double(), want.detach(), rtol=1e-5, atol=1e-4)
    assert float((dw.cpu().double() - dw64).abs().max()) <= 1e-5 * float(dw64.abs().max()) * 10
    assert float((ds.cpu().double() - ds64).abs().max()) <= 1e-5 * float(ds64.abs().max()) * 10


@pytest.mark.gpu
def test_captured_and_replayed(cuda):
    """Forward, backward and step captured into one graph and replayed with other inputs in the same buffers, eager work and
    synchronisations in between."""
    from building_gan_amd import ops
    V, D, n, S = 600, 64, 3000, 5
    ptr = torch.tensor([0, 10, 10, 900, 2500, 2900], dtype=torch.int32, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(0)

    def fill():
        ids.copy_(torch.randint(-1, V, (n,), generator=gen, device=cuda))
        w.copy_(torch.randn(V, 2 * D, generator=gen, device=cuda))
        g.copy_(torch.randn(n, D, generator=gen, device=cuda))
        dl.copy_(torch.randn(S, D, generator=gen, device=cuda))

    def passes():
        z = ops.embedding_raw(w, ids, 2.0)
        h, hl, heads = ops.gated_scan_raw(z[:, :D], z[:, D:], ptr, None, False, keep_heads=True)
        dx, dg, _ = ops.gated_scan_grad_raw(z[:, :D], z[:, D:], ptr, None, False, heads, g, dl)
        dw = ops.embedding_grad_raw(torch.cat([dx, dg], 1), ids, V, 2.0)
        hs, new = ops.gated_scan_step(z[:S, :D], z[:S, D:], hl)
        return z, h, hl, dx, dg, dw, hs, new

    ids = torch.zeros(n, dtype=torch.int64, device=cuda)
    w, g, dl = (torch.zeros(*s, device=cuda) for s in ((V, 2 * D), (n, D), (S, D)))
    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = passes()
    for k in range(4):
        fill()
        graph.replay()
        if k % 2:
            torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = passes()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (k, i)


@pytest.mark.gpu
def test_on_another_stream_and_two_calls_at_once(cuda):
    from building_gan_amd import ops
    c = scan_case(4000, 128, [0, 1000, 4000], torch.float32, 3)
    x, gate = c["x"].to(cuda).contiguous(), c["gate"].to(cuda).contiguous()
    ptr = torch.tensor([0, 1000, 4000], dtype=torch.int32, device=cuda)
    ids = torch.randint(0, 50, (4000,), device=cuda)
    want = ops.gated_scan(x, gate, ptr)[0]
    want_w = ops.embedding_grad_raw(x, ids, 50)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            outs.append((ops.gated_scan(x, gate, ptr)[0], ops.embedding_grad_raw(x, ids, 50)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, want_w) for a, b in outs)


# ------------------------------------------------------------------------------------------------ further sizes and calls
def test_pitches_past_32_bits_of_a_tile_are_refused():
    from building_gan_amd import _lib
    lib = _lib.load()
    p, far = 1 << 20, (1 << 21) + 1
    size = lib.bg_gated_scan_workspace(10, 8)
    fwd = lambda ldx, ldg, ldh: lib.bg_gated_scan_fwd(0, p, ldx, p, ldg, p, 2, 10, 8, None, 0, p, ldh, p, None, p, size, None)
    assert fwd(far, 8, 8) == -2 and fwd(8, far, 8) == -2 and fwd(8, 8, far) == -2
    bwd = lambda ldx, ldg, lddh, lddx, lddg: lib.bg_gated_scan_bwd(0, p, ldx, p, ldg, p, lddh, None, p, 2, 10, 8, None, 0, p, p, lddx, p, lddg,
                                                                   None, p, size, None)
    for k in range(5):
        assert bwd(*[far if i == k else 8 for i in range(5)]) == -2


def test_overlap_of_a_step_s_states():
    """Side by side in one buffer or the same rows: taken; anything else that shares memory: refused."""
    from building_gan_amd.ops import _shifted_overlap
    buf = torch.zeros(6, 24)
    a, b = buf[:, :12], buf[:, 12:]
    assert not _shifted_overlap(a, b) and not _shifted_overlap(b, a) and not _shifted_overlap(a, a)
    assert _shifted_overlap(buf[:, :13], buf[:, 11:24]) and _shifted_overlap(a[:4], a[1:5]) and _shifted_overlap(buf[:, 4:16], buf[:, :12])
    assert not _shifted_overlap(buf[:3], buf[3:]) and not _shifted_overlap(a, torch.zeros(6, 12))
    assert _shifted_overlap(buf[:1, :12], buf[:1, 6:18]) and not _shifted_overlap(buf[:1, :12], buf[:1, 12:])
    assert _shifted_overlap(a, buf.view(torch.float16)[:, :12])


@pytest.mark.gpu
def test_step_into_another_half_of_the_same_buffer(cuda):
    from building_gan_amd import _lib, ops
    buf, x = torch.randn(7, 64, device=cuda), torch.randn(7, 32, device=cuda)
    want = ops.gated_scan_step(x, x, buf[:, :32].contiguous())[1]
    keep = buf[:, :32].clone()
    ops.gated_scan_step(x, x, buf[:, :32], state_out=buf[:, 32:])
    assert torch.equal(buf[:, 32:], want) and torch.equal(buf[:, :32], keep)
    with pytest.raises(_lib.BganError):
        ops.gated_scan_step(x, x, buf[:, :32], state_out=buf[:, 16:48])
    with pytest.raises(_lib.BganError):
        ops.gated_scan_step(buf[:6, :32], x[:6], x[:6], state_out=buf[1:, :32])


# (4,096 is where one workgroup no longer sorts alone, 8,192 no border; the later ones: test_lookup_gradient_at_the_borders_of_the_sort)
@pytest.mark.gpu
@pytest.mark.parametrize("V,D,n,kind", [(7, 3, 5000, "uniform"), (20, 1, 999, "hot"), (5, 2, 70000, "missing"), (20, 132, 4097, "missing"),
                                        (21, 132, 4097, "missing"), (5000, 16, 4096, "uniform"), (5000, 16, 4097, "hot"),
                                        (900, 24, 8192, "uniform"), (900, 24, 8193, "missing"), (600, 2, 30000, "uniform")])
def test_lookup_at_the_borders_of_its_variants(cuda, V, D, n, kind):
    """Tables of a few rows with rows of less than a piece, and the token counts where the sort changes."""
    for dtype in (torch.float32, torch.bfloat16):
        w, ids, g = lookup_case(V, D, n, dtype, V * n + D, kind)
        check_lookup(cuda, w, ids, g, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse,dtype,ptr", [(False, torch.float32, [0, 16900]), (True, torch.float32, [0, 8200, 16900]),
                                               (False, torch.bfloat16, [0, 9000, 9001, 16900]), (True, torch.float16, [3, 16800])])
def test_scan_over_several_blocks_of_tiles(cuda, reverse, dtype, ptr):
    """More than 2 x 64 tiles of 128 rows: states handed from block to block, with and without a border in between."""
    c = scan_case(16900, 36, ptr, dtype, 21, slow=True)
    check_scan(cuda, c, ptr, reverse)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_many_segments_without_rows(cuda, reverse):
    """Their states pass through, in both directions, whatever the number of tiles."""
    from building_gan_amd import ops
    gen = torch.Generator().manual_seed(4)
    S, N = 20000, 700
    cuts = torch.randint(0, N + 1, (S - 1,), generator=gen).sort().values.tolist()
    ptr = torch.tensor([0] + cuts + [N], dtype=torch.int32)
    x, gate, h0 = torch.randn(N, 20, generator=gen), torch.randn(N, 20, generator=gen), torch.randn(S, 20, generator=gen)
    xs, gs, hs = (t.to(cuda).requires_grad_(True) for t in (x, gate, h0))
    h, hl = ops.gated_scan(xs, gs, ptr.to(cuda), hs, reverse)
    dl = torch.randn(S, 20, generator=gen)
    (d0,) = torch.autograd.grad(hl, hs, dl.to(cuda))
    none = (ptr[1:] == ptr[:-1])
    assert int(none.sum()) > S - N - 1
    assert torch.equal(hl.cpu()[none], h0[none]) and torch.equal(d0.cpu()[none], dl[none])
    some = torch.nonzero(~none).flatten().tolist()
    short = [int(ptr[s]) for s in some] + [N]
    h2, hl2 = ops.gated_scan(x.to(cuda), gate.to(cuda), torch.tensor(short, dtype=torch.int32, device=cuda), h0[some].to(cuda), reverse)
    assert torch.equal(h, h2) and torch.equal(hl[some], hl2)


@pytest.mark.gpu
def test_rows_past_2_31_elements(cuda):
    """The last rows of 2^31 and more elements (bf16, 4.3 GB a matrix): the same bits as a call on those rows alone."""
    from building_gan_amd import ops
    D, N0, n = 2048, 1 << 20, 300
    N = N0 + n
    gen = torch.Generator(device=cuda).manual_seed(6)
    x = torch.randn(N, D, generator=gen, device=cuda, dtype=torch.bfloat16)
    gate = torch.randn(N, D, generator=gen, device=cuda, dtype=torch.bfloat16)
    dh = torch.randn(N, D, generator=gen, device=cuda, dtype=torch.bfloat16)
    ptr = torch.tensor([0, N0, N], dtype=torch.int32, device=cuda)           # N0 is a border of 64 tiles: joined alike
    h, hl, heads = ops.gated_scan_raw(x, gate, ptr, None, False, keep_heads=True)
    own, ownl, own_heads = ops.gated_scan_raw(x[N0:], gate[N0:], 1, None, False, keep_heads=True)
    assert torch.equal(h[N0:], own) and torch.equal(hl[1:], ownl)
    dx, dg, _ = ops.gated_scan_grad_raw(x, gate, ptr, None, False, heads, dh, None, False)
    odx, odg, _ = ops.gated_scan_grad_raw(x[N0:], gate[N0:], 1, None, False, own_heads, dh[N0:], None, False)
    assert torch.equal(dx[N0:], odx) and torch.equal(dg[N0:], odg)
    del h, heads, dx, dg, gate, dh
    ids = torch.randint(0, 50, (N,), generator=gen, device=cuda)
    w = torch.randn(50, D, generator=gen, device=cuda, dtype=torch.bfloat16)
    out = ops.embedding(w, ids)                                              # (stored around the caches)
    assert torch.equal(out[N0:], w[ids[N0:]]) and torch.equal(out[:n], w[ids[:n]])
    del out
    ids[:N0] = -1
    g = x.sign()                                                             # sums of +-1: exact in any order
    want = torch.zeros(50, D, device=cuda).index_add_(0, ids[N0:], g[N0:].float())
    assert torch.equal(ops.embedding_grad_raw(g, ids, 50).float(), want)
    assert torch.equal(ops.embedding_grad_raw(g[:, :24], ids % 7 - (ids < 0).long() * 9, 20)[:7].float(),
                       torch.zeros(7, 24, device=cuda).index_add_(0, ids[N0:] % 7, g[N0:, :24].float()))


@pytest.mark.gpu
def test_autograd_captured_and_replayed(cuda):
    """A step of training, forward and backward through autograd, captured once and replayed on changing inputs."""
    from building_gan_amd import ops
    B, T, V, D = 3, 150, 40, 48
    gen = torch.Generator(device=cuda).manual_seed(1)
    w = torch.randn(V, 2 * D, generator=gen, device=cuda).requires_grad_(True)
    h0 = torch.randn(B, D, generator=gen, device=cuda).requires_grad_(True)
    ids = torch.zeros(B, T, dtype=torch.int64, device=cuda)
    cot = torch.zeros(B, T, D, device=cuda)

    def step():
        z = ops.embedding(w, ids, 0.5)
        h, hl = ops.gated_scan(z[..., :D], z[..., D:], h0=h0, reverse=True)
        grads = torch.autograd.grad((h, hl), (w, h0), (cot, h0.detach()))
        return (h.detach(), hl.detach()) + grads             # (no graph of these leaves lives on)

    def fill():
        ids.copy_(torch.randint(-1, V, (B, T), generator=gen, device=cuda))
        cot.copy_(torch.randn(B, T, D, generator=gen, device=cuda))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        fill()
        graph.replay()
        if k % 2:
            torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for i, (a, b) in enumerate(zip(got, step())):
            assert torch.equal(a, b), (k, i)


@pytest.mark.gpu
def test_one_token_and_broadcast_operands(cuda):
    """A scalar id, no ids with a gradient asked for, and operands expanded over the batch: their gradients add up."""
    from building_gan_amd import ops
    w = torch.randn(6, 9, device=cuda, requires_grad=True)
    one = ops.embedding(w, torch.tensor(4, device=cuda), 2.0)
    assert one.shape == (9,) and torch.equal(torch.autograd.grad(one, w, torch.ones(9, device=cuda))[0][:, 0].cpu(), torch.tensor([0., 0, 0, 0, 2, 0]))
    none = ops.embedding(w, torch.zeros(0, 3, dtype=torch.int64, device=cuda))
    assert not torch.autograd.grad(none, w, torch.zeros(0, 3, 9, device=cuda))[0].any()
    x = torch.randn(1, 40, 12, device=cuda, requires_grad=True)
    gate = torch.randn(3, 40, 12, device=cuda, requires_grad=True)
    h, hl = ops.gated_scan(x.expand(3, 40, 12), gate)
    dx, dg = torch.autograd.grad(h.sum() + hl.sum(), (x, gate))
    xs = x.detach().expand(3, 40, 12).contiguous().requires_grad_(True)
    h2, hl2 = ops.gated_scan(xs, gate)
    dx2, dg2 = torch.autograd.grad(h2.sum() + hl2.sum(), (xs, gate))
    assert torch.equal(h, h2) and torch.equal(dg, dg2) and torch.equal(dx, dx2.sum(0, keepdim=True))
    y = torch.randn(50, 8, device=cuda, requires_grad=True)              # one tensor as both operands
    (dy,) = torch.autograd.grad(ops.gated_scan(y, y)[0].sum(), y)
    y1, y2 = y.detach().clone().requires_grad_(True), y.detach().clone().requires_grad_(True)
    a, b = torch.autograd.grad(ops.gated_scan(y1, y2)[0].sum(), (y1, y2))
    assert torch.equal(dy, a + b)


@pytest.mark.gpu
def test_two_captured_graphs_replayed_at_once(cuda):
    """Each graph keeps its own workspaces: replays on two streams, at the same time, do not disturb each other."""
    from building_gan_amd import ops
    gen = torch.Generator(device=cuda).manual_seed(12)
    sides = []
    for k, (N, D, V) in enumerate(((20000, 128, 900), (15000, 200, 40))):
        x, gate, dh = (torch.randn(N, D, generator=gen, device=cuda) for _ in range(3))
        ids = torch.randint(-1, V, (N,), generator=gen, device=cuda)
        ptr = torch.tensor([0, N // 3, N], dtype=torch.int32, device=cuda)

        def passes(x=x, gate=gate, dh=dh, ids=ids, ptr=ptr, V=V, k=k):
            h, last, heads = ops.gated_scan_raw(x, gate, ptr, None, k == 1, keep_heads=True)
            dx, dg, _ = ops.gated_scan_grad_raw(x, gate, ptr, None, k == 1, heads, dh, None)
            return h, last, dx, dg, ops.embedding_grad_raw(dx, ids, V)

        want = passes()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = passes()
        sides.append((graph, outs, want, torch.cuda.Stream(), passes))       # (passes holds what the graph reads)
    for r in range(4):
        for _, outs, *_ in sides:
            for t in outs:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for k, (_, outs, want, *_) in enumerate(sides):
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), (r, k)


# ------------------------------------------------------------------------------------------------ autograd around the calls
@pytest.fixture
def no_launch(monkeypatch):
    """The wrappers on CPU tensors with every launch left out (results are whatever the memory held): what they do before and
    after one.  Returns the list of the calls made, as (entry point, arguments)."""
    from building_gan_amd import _lib, ops
    real, calls = _lib.load(), []

    class Library:
        def __getattr__(self, name):
            if name in _lib._SIZES:
                return getattr(real, name)
            return lambda *a: calls.append((name, a)) or 0

    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(_lib, "require_device", lambda *a: None)
    monkeypatch.setattr(_lib, "elsewhere", lambda t: False)
    monkeypatch.setattr(ops, "stream", lambda: 0)
    return calls


def step_in_place_before_the_backward_pass(dev):
    """States that a scan's backward pass will read are overwritten by a step: autograd has to notice."""
    from building_gan_amd import ops
    x = torch.ones(4, 8, device=dev, requires_grad=True)
    state = torch.zeros(2, 8, device=dev)
    h, _ = ops.gated_scan(x, torch.zeros(4, 8, device=dev), torch.tensor([0, 1, 4], dtype=torch.int32, device=dev), state)
    row = torch.ones(2, 8, device=dev)
    seen = state._version
    ops.gated_scan_step(row, row, torch.zeros(2, 8, device=dev))             # states of its own: nothing of ours changes
    assert state._version == seen
    ops.gated_scan_step(row, row, state, state_out=state)
    assert state._version > seen
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    buf = torch.zeros(2, 24, device=dev)                                     # a view's base knows too
    ops.gated_scan_step(row, row, torch.zeros(2, 8, device=dev), state_out=buf[:, 8:16])
    assert buf._version > 0
    with torch.inference_mode():
        kept = torch.zeros(2, 8, device=dev)
        assert ops.gated_scan_step(row, row, kept, state_out=kept)[1] is kept


def test_step_in_place_is_seen_by_autograd(no_launch):
    step_in_place_before_the_backward_pass(torch.device("cpu"))


@pytest.mark.gpu
def test_step_in_place_is_seen_by_autograd_on_the_gpu(cuda):
    step_in_place_before_the_backward_pass(cuda)


def steps_that_would_lose_a_gradient(dev):
    from building_gan_amd import _lib, ops
    plain = lambda: torch.zeros(3, 8, device=dev)
    wants = lambda: torch.zeros(3, 8, device=dev, requires_grad=True)
    for call in (lambda: ops.gated_scan_step(wants(), plain(), plain()), lambda: ops.gated_scan_step(plain(), wants(), plain()),
                 lambda: ops.gated_scan_step(plain(), plain(), wants()),
                 lambda: ops.gated_scan_step(plain(), plain(), plain(), state_out=wants())):
        with pytest.raises(_lib.BganError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    kept = wants()
    with torch.no_grad():
        assert ops.gated_scan_step(plain(), plain(), kept, state_out=kept)[1] is kept
    assert not ops.gated_scan_step(wants().detach(), plain(), plain())[0].requires_grad


def test_step_refuses_operands_that_want_a_gradient(no_launch):
    steps_that_would_lose_a_gradient(torch.device("cpu"))


@pytest.mark.gpu
def test_step_refuses_operands_that_want_a_gradient_on_the_gpu(cuda):
    steps_that_would_lose_a_gradient(cuda)


def forward_mode_calls(dev):
    """Forward-mode derivatives are not offered: an operand's tangent is an error, never a result without one."""
    import torch.autograd.forward_ad as fw
    from building_gan_amd import ops
    w, ids, h0 = torch.ones(4, 8, device=dev), torch.tensor([0, 3], device=dev), torch.zeros(1, 8, device=dev)
    with fw.dual_level():
        d, d0 = fw.make_dual(w, torch.ones_like(w)), fw.make_dual(h0, torch.ones_like(h0))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: ops.embedding(d, ids), lambda: ops.gated_scan(d, w), lambda: ops.gated_scan(w, d),
                             lambda: ops.gated_scan(w, w, None, d0), lambda: ops.gated_scan(d.view(2, 2, 8), w.view(2, 2, 8))):
                    with pytest.raises(RuntimeError):
                        call()
                assert ops.embedding(w, ids).shape == (2, 8) and ops.gated_scan(w, w, None, h0)[0].shape == (4, 8)     # no tangent


def test_operands_with_tangents_are_refused(no_launch):
    forward_mode_calls(torch.device("cpu"))


@pytest.mark.gpu
def test_operands_with_tangents_are_refused_on_the_gpu(cuda):
    forward_mode_calls(cuda)


def forward_over_reverse(dev):
    """The cotangent of a backward pass may carry a tangent too (a Hessian's product with a vector taken that way)."""
    import torch.autograd.forward_ad as fw
    from building_gan_amd import ops
    w, ids = torch.ones(4, 8, device=dev, requires_grad=True), torch.tensor([0, 3], device=dev)
    dual = lambda *s: fw.make_dual(torch.ones(*s, device=dev), torch.ones(*s, device=dev))
    with fw.dual_level():
        out = ops.embedding(w, ids)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, w, dual(2, 8), retain_graph=True)
        assert torch.autograd.grad(out, w, torch.ones(2, 8, device=dev))[0].shape == (4, 8)
        h, last = ops.gated_scan(w, w.detach())
        for outs, grads in ((h, dual(4, 8)), (last, dual(1, 8)), ((h, last), (torch.ones(4, 8, device=dev), dual(1, 8)))):
            with pytest.raises(RuntimeError):
                torch.autograd.grad(outs, w, grads, retain_graph=True)
        assert torch.autograd.grad((h, last), w, (torch.ones(4, 8, device=dev), torch.ones(1, 8, device=dev)))[0].shape == (4, 8)


def test_cotangents_with_tangents_are_refused(no_launch):
    forward_over_reverse(torch.device("cpu"))


@pytest.mark.gpu
def test_cotangents_with_tangents_are_refused_on_the_gpu(cuda):
    forward_over_reverse(cuda)


def test_overlap_of_a_step_s_state_and_rows(no_launch):
    """The states may be written where they stand, an operand's rows may not; and the pitch of a single row means nothing."""
    from building_gan_amd import _lib, ops
    x, gate, state = torch.zeros(3, 8), torch.zeros(3, 8), torch.zeros(3, 8)
    for out in (x, gate):
        with pytest.raises(_lib.BganError, match="shares memory"):
            ops.gated_scan_step(x, gate, state, state_out=out)
    for same in (x, gate):                                                   # written as states, read as rows
        with pytest.raises(_lib.BganError, match="shares memory"):
            ops.gated_scan_step(x, gate, same, state_out=same)
    assert ops.gated_scan_step(x, gate, state, state_out=state)[1] is state
    buf = torch.zeros(2, 32)
    row, again = buf[:1, :16], buf.as_strided((1, 16), (16, 1))              # the same row, told in two ways
    assert row.stride() != again.stride()
    one = torch.zeros(1, 16)
    ops.gated_scan_step(one, one, row, state_out=again)
    ops.gated_scan_step(one, one, again, state_out=row)
    with pytest.raises(_lib.BganError, match="shares memory"):
        ops.gated_scan_step(one, one, row, state_out=buf.as_strided((1, 16), (16, 1), 8))
    with pytest.raises(_lib.BganError, match="shares memory"):
        ops.gated_scan_step(again, one, one, state_out=row)
    tall = buf.view(64, 1)                                                   # a single column: its inner stride means nothing
    ops.gated_scan_step(torch.zeros(64, 1), torch.zeros(64, 1), tall, state_out=buf.as_strided((64, 1), (1, 7)))


def far_rows(dev, n=5, D=8, pitch=(1 << 21) + 4):
    buf = torch.zeros(n, pitch, device=dev)
    gen = torch.Generator().manual_seed(0)
    for k in (0, D, 2 * D):
        buf[:, k:k + D] = torch.randn(n, D, generator=gen).to(dev)
    return buf[:, :D], buf[:, D:2 * D], buf[:, 2 * D:3 * D]


def test_far_rows_are_copied_before_a_scan(no_launch):
    """Rows farther apart than a tile's 32-bit offsets reach: the entry points refuse such a pitch, so the wrappers copy."""
    from building_gan_amd import ops
    x, gate, dh = far_rows(torch.device("cpu"))
    x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    h, _ = ops.gated_scan(x, gate)
    torch.autograd.grad(h, (x, gate), dh)
    ops.gated_scan_grad_raw(x.detach(), gate.detach(), 1, None, False, torch.zeros(ops._scan_sizes(5, 8)[0]), dh, None)
    (f, fa), (b, ba), (r, ra) = no_launch
    assert f == "bg_gated_scan_fwd" and b == r == "bg_gated_scan_bwd"
    assert [fa[2], fa[4]] == [8, 8] and [ba[2], ba[4], ba[6]] == [ra[2], ra[4], ra[6]] == [8, 8, 8]      # the pitches


@pytest.mark.gpu
def test_far_rows_are_scanned(cuda):
    from building_gan_amd import ops
    x, gate, dh = far_rows(cuda)
    near = [t.contiguous() for t in (x, gate, dh)]
    out = []
    for xx, gg, dd in ((x, gate, dh), near):
        xx, gg = xx.detach().requires_grad_(True), gg.detach().requires_grad_(True)
        h, last = ops.gated_scan(xx, gg)
        out.append((h, last) + torch.autograd.grad(h, (xx, gg), dd))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    state = torch.zeros(5, 8, device=cuda)
    assert torch.equal(ops.gated_scan_step(x, gate, state)[1], ops.gated_scan_step(near[0], near[1], state)[1])
    ids = torch.tensor([0, 4, 2, 1, 3], device=cuda)
    assert torch.equal(ops.embedding(x, ids), near[0][ids])
    assert torch.equal(ops.embedding_grad_raw(x, ids, 30), ops.embedding_grad_raw(near[0], ids, 30))


# ------------------------------------------------------------------------------------------------ every variant of the sort, equal segments
@pytest.mark.gpu
@pytest.mark.parametrize("ids_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("V", [21, 700, 300000])                                 # one, two and three passes over the keys
@pytest.mark.parametrize("n", [4096, 4097, 65536, 65537, 131072, 131073, 200001, 262144, 262145])
def test_lookup_gradient_at_the_borders_of_the_sort(cuda, n, V, ids_dtype):
    """Token counts at which the sort takes another form: one workgroup; 2, 4 and 8 keys a lane; the tiles' counts added up by
    every workgroup, and scanned from 64 tiles on.  Sums of small whole numbers: exact in any order."""
    from building_gan_amd import ops
    gen = torch.Generator().manual_seed(n + V)
    ids = torch.randint(0, V, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < 0.3] = V // 3                         # a run over many tiles of slots
    ids[torch.rand(n, generator=gen) < 0.1] = -1
    ids[0], ids[n - 1], ids[n // 2] = V - 1, V - 1, V                        # the ends of the order, a missing token
    g = torch.randint(-3, 4, (n, 8), generator=gen).float()
    there = (ids >= 0) & (ids < V)
    want = torch.zeros(V, 8, dtype=torch.float64).index_add_(0, ids[there], g[there].double()) * 0.5
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.embedding_grad_raw(g.to(cuda).to(dtype), ids.to(cuda).to(ids_dtype), V, 0.5)
        assert torch.equal(got.cpu(), want.to(dtype)), (dtype, int((got.cpu() != want.to(dtype)).sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("B,T,D", [(6, 77, 24), (1, 300, 12), (40, 1, 8), (3, 1001, 68), (9, 128, 64)])
def test_scan_of_a_batch_and_its_gradients(cuda, B, T, D, reverse, dtype):
    """[B, T, D] has no row pointer: values and gradients against float64 through the row pointer, and bit for bit alike."""
    from building_gan_amd import ops
    ptr = list(range(0, B * T + 1, T))
    c = scan_case(B * T, D, ptr, dtype, B + T)
    want = check_scan(cuda, c, ptr, reverse)
    z, h0 = c["z"].to(cuda).view(B, T, 2 * D).requires_grad_(True), c["h0"].to(cuda).requires_grad_(True)
    h, last = ops.gated_scan(z[..., :D], z[..., D:], None, h0, reverse)
    dz, d0 = torch.autograd.grad((h, last), (z, h0), (c["dh"].to(cuda).view(B, T, D), c["dlast"].to(cuda)))
    got = (h.reshape(B * T, D), last, dz[..., :D].reshape(B * T, D), dz[..., D:].reshape(B * T, D), d0)
    for name, a, b in zip(("h", "h_last", "dx", "dgate", "dh0"), got, want):
        assert torch.equal(a, b), name


# ------------------------------------------------------------------------------------------------ calls the limits and the header allow
@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_at_the_largest_pitch(cuda, dtype, reverse):
    """Rows 2^21 elements apart, in tiles of 512 rows: offsets in a tile up to 4 * 511 * 2^21 bytes, just under 2^32."""
    from building_gan_amd import ops
    N, D, P = 530, 16, 1 << 21
    gen = torch.Generator().manual_seed(3)
    near = [torch.randn(N, D, generator=gen).to(dtype).to(cuda) for _ in range(3)]
    buf = torch.empty(N, P, dtype=dtype, device=cuda)
    far = [buf[:, 16 * k:16 * k + D] for k in range(3)]
    for a, b in zip(far, near):
        a.copy_(b)
    ptr = torch.tensor([0, 100, 519, 530], dtype=torch.int32, device=cuda)
    outs = []
    for x, gate, dh in (far, near):
        h, last, heads = ops.gated_scan_raw(x, gate, ptr, None, reverse, keep_heads=True)
        outs.append((h, last) + ops.gated_scan_grad_raw(x, gate, ptr, None, reverse, heads, dh, None))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_widest_rows(cuda, dtype):
    """2^15 columns of a table, by few rows and sorted, and 2^20 columns of a scan."""
    from building_gan_amd import ops
    gen = torch.Generator().manual_seed(1)
    for V in (20, 23):
        w = torch.randint(-4, 5, (V, 1 << 15), generator=gen).to(dtype).to(cuda)
        ids = torch.randint(-1, V + 1, (37,), generator=gen)
        g = torch.randint(-4, 5, (37, 1 << 15), generator=gen).to(dtype).to(cuda)
        there = (ids >= 0) & (ids < V)
        want = torch.zeros(37, 1 << 15, dtype=dtype)
        want[there] = w.cpu()[ids[there]]
        assert torch.equal(ops.embedding(w, ids.to(cuda)).cpu(), want)
        want = torch.zeros(V, 1 << 15).index_add_(0, ids[there], g.cpu()[there].float()).to(dtype)
        assert torch.equal(ops.embedding_grad_raw(g, ids.to(cuda), V).cpu(), want)
    D = 1 << 20
    x, gate = (torch.randn(5, D, generator=gen).to(dtype).to(cuda) for _ in range(2))
    h, last = ops.gated_scan(x, gate, torch.tensor([0, 3, 5], dtype=torch.int32, device=cuda))
    for cols in (slice(0, 64), slice(D - 64, D)):
        c, cl = ops.gated_scan(x[:, cols], gate[:, cols], torch.tensor([0, 3, 5], dtype=torch.int32, device=cuda))
        assert torch.equal(h[:, cols], c) and torch.equal(last[:, cols], cl)
    s, new = ops.gated_scan_step(x, gate, torch.ones(5, D, device=cuda))
    c, cn = ops.gated_scan_step(x[:, -64:], gate[:, -64:], torch.ones(5, 64, device=cuda))
    assert torch.equal(s[:, -64:], c) and torch.equal(new[:, -64:], cn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [3, 33, 64, 130])
def test_pitched_outputs_of_the_entry_points(cuda, D, dtype):
    """Outputs with a row pitch, which only the C entry points offer: the same bits, and nothing between the rows is written."""
    from building_gan_amd import _lib, ops
    lib, s = _lib.load(), _lib.stream()
    code, N, P = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], 700, D + 5
    ptr = [0, 0, 1, 300, 690]
    c = scan_case(N, D, ptr, dtype, D)
    x, gate, h0, dh, dl = c["x"].to(cuda).contiguous(), c["gate"].to(cuda).contiguous(), c["h0"].to(cuda), c["dh"].to(cuda), c["dlast"].to(cuda)
    rp = torch.tensor(ptr, dtype=torch.int32, device=cuda)
    size = lib.bg_gated_scan_workspace(N, D)
    ws = torch.empty(size, dtype=torch.uint8, device=cuda)

    def out(n):                                              # rows D wide, one element off the buffer's start, all sevens
        buf = torch.full((n * P + 8,), 7.0, dtype=dtype, device=cuda)
        return buf, buf[1:1 + n * P].view(n, P)[:, :D]

    def rest_is_seven(buf, view):
        view.fill_(7.0)
        return bool((buf == 7.0).all())

    for rev in (0, 1):
        h, last, heads = ops.gated_scan_raw(x, gate, rp, h0, bool(rev), keep_heads=True)
        dx, dg, d0 = ops.gated_scan_grad_raw(x, gate, rp, h0, bool(rev), heads, dh, dl)
        (b1, v1), (b2, v2), (b3, v3) = out(N), out(N), out(N)
        assert lib.bg_gated_scan_fwd(code, x.data_ptr(), D, gate.data_ptr(), D, rp.data_ptr(), 4, N, D, h0.data_ptr(), rev, v1.data_ptr(), P,
                                     None, None, ws.data_ptr(), size, s) == 0                        # without h_last and heads
        assert lib.bg_gated_scan_bwd(code, x.data_ptr(), D, gate.data_ptr(), D, dh.data_ptr(), D, dl.data_ptr(), rp.data_ptr(), 4, N, D,
                                     h0.data_ptr(), rev, heads.data_ptr(), v2.data_ptr(), P, v3.data_ptr(), P, None, ws.data_ptr(), size, s) == 0
        assert torch.equal(v1, h) and torch.equal(v2, dx) and torch.equal(v3, dg)
        assert rest_is_seven(b1, v1) and rest_is_seven(b2, v2) and rest_is_seven(b3, v3)
    state = torch.randn(N, D, device=cuda)
    want, new = ops.gated_scan_step(x, gate, state)
    b, v = out(N)
    assert lib.bg_gated_scan_step(code, x.data_ptr(), D, gate.data_ptr(), D, state.data_ptr(), D, N, D, v.data_ptr(), P, state.data_ptr(), D, s) == 0
    assert torch.equal(v, want) and torch.equal(state, new) and rest_is_seven(b, v)
    ids = torch.randint(-1, N, (N,), device=cuda)
    b, v = out(N)
    assert lib.bg_embedding_fwd(code, x.data_ptr(), D, N, ids.data_ptr(), 1, N, D, 2.0, v.data_ptr(), P, s) == 0
    assert torch.equal(v, ops.embedding(x, ids, 2.0)) and rest_is_seven(b, v)


@pytest.mark.gpu
@pytest.mark.parametrize("reverse", [False, True])
def test_row_pointers_past_the_rows_end_there(cuda, reverse):
    """Entries outside [0, rows] count as the nearer end."""
    c = scan_case(460, 20, [0, 100, 460, 460], torch.float32, 5)
    a = check_scan(cuda, c, [0, 100, 460, 460], reverse)
    b = check_scan_values(cuda, c, [-7, 100, 461, 2 ** 31 - 1], reverse)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def check_scan_values(cuda, c, ptr, reverse):
    from building_gan_amd import ops
    x, gate, h0 = (c[k].to(cuda).requires_grad_(True) for k in ("x", "gate", "h0"))
    h, hl = ops.gated_scan(x, gate, torch.tensor(ptr, dtype=torch.int32, device=cuda), h0, reverse)
    return (h, hl) + torch.autograd.grad((h, hl), (x, gate, h0), (c["dh"].to(cuda), c["dlast"].to(cuda)))


@pytest.mark.gpu
def test_small_tables_captured_and_replayed(cuda):
    """The sums of tables of up to 20 rows (above 16 they ask for more LDS than a kernel has by itself), no tokens, one-workgroup
    and many-workgroup sorts: captured, and replayed on changing inputs."""
    from building_gan_amd import ops
    cases = [(7, 24, 900), (17, 130, 5000), (20, 3, 4000), (20, 64, 0), (300, 64, 0), (300, 33, 4000), (90000, 8, 9000)]
    gen = torch.Generator(device=cuda).manual_seed(4)
    ids = [torch.zeros(n, dtype=torch.int32, device=cuda) for _, _, n in cases]
    g = [torch.zeros(n, D, device=cuda) for _, D, n in cases]

    def fill():
        for (V, _, n), i, gg in zip(cases, ids, g):
            if n:
                i.copy_(torch.randint(-1, V + 1, (n,), generator=gen, device=cuda))
                gg.copy_(torch.randn(gg.shape, generator=gen, device=cuda))

    def passes():
        return [ops.embedding_grad_raw(gg, i, V, 0.5) for (V, _, _), i, gg in zip(cases, ids, g)]

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = passes()
    for k in range(4):
        fill()
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        if k % 2:
            torch.cuda.synchronize()
        for a, b in zip([t.clone() for t in outs], passes()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensors_kept_elsewhere_and_a_graph_used_twice(cuda):
    """Operands saved on the host and brought back, one backward pass run twice over a kept graph, a checkpointed call: the same
    gradients; an operand changed in between is an error."""
    from torch.utils.checkpoint import checkpoint
    from building_gan_amd import ops
    ptr = torch.tensor([0, 33, 200], dtype=torch.int32, device=cuda)
    z = torch.randn(200, 40, device=cuda, requires_grad=True)
    h0 = torch.randn(2, 20, device=cuda, requires_grad=True)
    w = torch.randn(30, 40, device=cuda, requires_grad=True)
    ids = torch.randint(0, 30, (200,), device=cuda)

    def f(z, h0, w):
        y = ops.embedding(w, ids) + z
        h, last = ops.gated_scan(y[:, :20], y[:, 20:], ptr, h0)
        return (h * h).sum() + last.sum()

    loss = f(z, h0, w)
    want = torch.autograd.grad(loss, (z, h0, w), retain_graph=True)
    again = torch.autograd.grad(loss, (z, h0, w))
    with torch.autograd.graph.save_on_cpu():
        loss = f(z, h0, w)
    host = torch.autograd.grad(loss, (z, h0, w))
    ck = torch.autograd.grad(checkpoint(f, z, h0, w, use_reentrant=False), (z, h0, w))
    for got in (again, host, ck):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, gate = torch.randn(50, 8, device=cuda), torch.randn(50, 8, device=cuda, requires_grad=True)
    h, _ = ops.gated_scan(x, gate)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
