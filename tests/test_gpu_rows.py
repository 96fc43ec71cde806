"""The row lookup (binned.gather_rows) and its gradients against float64, at the sizes, masks and layouts
where they can go wrong.

Tolerances, with u = 2^-24 the fp32 rounding and r = finfo(type).eps / 2 that of the result:
* out = round(round(scale w) t): the factor, the product and the result, 2u + r relative (r = u for fp32);
* a gradient row adds n products of a rounded factor: each term is off by 3u (factor, product, weight
  as given), each of the n adds by u of the running sum of magnitudes: (n + 3) u sum|f g| + r |value|;
* a weight's gradient adds C products: (C + 3) u |scale| sum|g t|.
fp16 results below the normal range are off by half the smallest step (2^-25) instead.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(R, C, shape, dt=torch.float32, seed=0, index=torch.int64, unused=0.2, hot=0.0, valid=True, weight=True):
    g = torch.Generator().manual_seed(seed)
    N = 1
    for s in shape:
        N *= s
    idx = torch.randint(0, max(R, 1), (N,), generator=g)
    idx[torch.rand(N, generator=g) < hot] = R // 2          # one row with most of the uses
    idx[torch.rand(N, generator=g) < unused / 2] = -1
    ok = torch.rand(N, generator=g) >= unused / 2
    if R == 0:
        idx.fill_(-1)
    return dict(table=torch.randn(R, C, generator=g).to(dt).to(DEV), idx=idx.to(index).reshape(shape).to(DEV),
                valid=ok.reshape(shape).to(DEV) if valid else None,
                weight=(torch.rand(N, generator=g) * 2 - 0.5).reshape(shape).to(DEV) if weight else None,
                gout=torch.randn(N, C, generator=g).to(dt).reshape(*shape, C).to(DEV))


def _check(x, scale=1.0, gout=None):
    from tt_splat_b200 import binned
    table = x["table"].detach().requires_grad_(True)
    weight = None if x["weight"] is None else x["weight"].detach().requires_grad_(True)
    out = binned.gather_rows(table, x["idx"], valid=x["valid"], weight=weight, scale=scale)
    gout = x["gout"] if gout is None else gout
    grads = torch.autograd.grad(out, [table] + ([weight] if weight is not None else []), gout)
    dt, (R, C) = table.dtype, table.shape
    r, sub = torch.finfo(dt).eps / 2, (2.0 ** -25 if dt == torch.float16 else 0.0)
    idx = x["idx"].reshape(-1).long()
    use = idx >= 0 if x["valid"] is None else (idx >= 0) & x["valid"].reshape(-1)
    f = torch.full(idx.shape, float(scale), dtype=torch.float64, device=DEV)
    if weight is not None:
        f = f * weight.detach().reshape(-1).double()
    t64, n = table.detach().double(), use.nonzero()[:, 0]
    ref = torch.zeros(idx.numel(), C, dtype=torch.float64, device=DEV)
    ref[n] = f[n, None] * t64[idx[n]]
    assert out.shape == (*x["idx"].shape, C) and out.dtype == dt
    err = (out.detach().reshape(-1, C).double() - ref).abs()
    assert (err <= ref.abs() * (r + 2.5 * U) + sub).all()
    assert (out.detach().reshape(-1, C)[~use] == 0).all()

    go = gout.reshape(-1, C).double()
    term = f[n, None] * go[n]
    gt = torch.zeros(R, C, dtype=torch.float64, device=DEV).index_add_(0, idx[n], term)
    mag = torch.zeros(R, C, dtype=torch.float64, device=DEV).index_add_(0, idx[n], term.abs())
    cnt = torch.bincount(idx[n], minlength=R)[:R, None]
    assert grads[0].shape == table.shape and grads[0].dtype == dt
    err = (grads[0].double() - gt).abs()
    assert (err <= (cnt + 3) * U * mag * 1.01 + (r + U) * gt.abs() + sub).all()
    assert (grads[0][cnt[:, 0] == 0] == 0).all()
    if weight is not None:
        dots = go[n] * t64[idx[n]]
        gw, gm = torch.zeros_like(f), torch.zeros_like(f)
        gw[n], gm[n] = scale * dots.sum(1), abs(scale) * dots.abs().sum(1)
        assert grads[1].shape == weight.shape and grads[1].dtype == torch.float32
        err = (grads[1].reshape(-1).double() - gw).abs()
        assert (err <= (C + 3) * U * gm * 1.01).all()
        assert (grads[1].reshape(-1)[~use] == 0).all()
    return out, grads


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", [1, 2, 3, 4, 7, 8, 12, 16, 31, 33, 45, 64, 100, 256, 1000, 2049])
def test_widths(C, dt):
    _check(_inputs(37, C, (129,), dt, seed=C), scale=0.75)


def test_the_widest_rows():
    """Rows of more column parts than any other test has, and the widest there are."""
    for C in (2 ** 21 + 1, 2 ** 22):
        _check(_inputs(3, C, (5,), seed=1, weight=False))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 255, 257, 4095, 4097, 8193, 40000])
def test_lengths(N, dt):
    _check(_inputs(300, 13, (N,), dt, seed=N, index=torch.int32))


@pytest.mark.parametrize("R", [1, 2, 255, 256, 257, 65535, 65536, 65537, 300000, 17000000])
def test_table_sizes(R):
    """Row counts on both sides of the sort's digits; the last and first row are looked up."""
    x = _inputs(R, 2, (20000,), seed=R % 1000)
    x["idx"][0], x["idx"][1] = R - 1, 0
    x["valid"][:2] = True
    _check(x)


@pytest.mark.parametrize("hot", [0.5, 0.99, 1.0])
@pytest.mark.parametrize("N,C", [(5000, 45), (100000, 6), (70000, 128)])
def test_row_with_most_uses(hot, N, C):
    _check(_inputs(1000, C, (N,), torch.bfloat16, seed=N, hot=hot))


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", [3, 11, 21, 31, 45, 63, 125])
def test_many_lookups_of_odd_rows(C, dt, weight):
    """Rows packed several units to a lane, in the longest chunks."""
    _check(_inputs(4000, C, (300001,), dt, seed=C, hot=0.1, weight=weight))


@pytest.mark.parametrize("valid,weight", [(False, False), (True, False), (False, True)])
def test_without_mask_or_weight(valid, weight):
    _check(_inputs(50, 9, (40, 16), seed=3, valid=valid, weight=weight), scale=-3.5)


def test_nothing_looked_up():
    from tt_splat_b200 import binned
    x = _inputs(20, 5, (64,), unused=0.0)
    x["valid"][:] = False
    _check(x)
    x["valid"][:] = True
    x["idx"][:] = -7
    _check(x)
    _check(_inputs(0, 5, (64,)))                                       # a table without rows
    t = torch.randn(20, 5, device=DEV, requires_grad=True)
    out = binned.gather_rows(t, torch.empty(0, 3, dtype=torch.int32, device=DEV))
    assert out.shape == (0, 3, 5)
    assert (torch.autograd.grad(out, t, torch.empty_like(out))[0] == 0).all()
    t = torch.randn(20, 0, device=DEV, requires_grad=True)
    out = binned.gather_rows(t, torch.zeros(4, dtype=torch.int32, device=DEV))
    assert out.shape == (4, 0) and torch.autograd.grad(out, t, out.detach())[0].shape == (20, 0)


def test_shapes_of_tables_and_indices():
    from tt_splat_b200 import binned
    t = torch.randn(30, 15, 3, device=DEV)
    i = torch.randint(0, 30, (2, 4, 8), device=DEV)
    assert torch.equal(binned.gather_rows(t, i), t[i])
    v = torch.randn(30, device=DEV)
    assert torch.equal(binned.gather_rows(v, i), v[i])
    assert torch.equal(binned.gather_rows(t, i[0, 0, 0]), t[i[0, 0, 0]])
    assert torch.equal(binned.gather_rows(t, i.transpose(0, 2)), t[i.transpose(0, 2)])


@pytest.mark.parametrize("rows,index", [((30,), (4, 8)), ((30,), (30, 1)), ((30, 1), (5, 3)), ((30, 2, 3), (7,)), ((30, 15, 3), (2, 4, 8)),
                                        ((30, 6), ()), ((30,), ()), ((30, 4), (20, 500))])
def test_gradients_of_any_shape(rows, index):
    """Against index_add in float64 of flattened rows, (n + 3) u sum|g| for a row of n uses."""
    from tt_splat_b200 import binned
    t = torch.randn(rows, device=DEV, requires_grad=True)
    i = torch.randint(0, 30, index, device=DEV)
    out = binned.gather_rows(t, i)
    assert out.shape == (*index, *rows[1:]) and torch.equal(out, t.detach()[i])
    gout = torch.randn(out.shape, device=DEV)
    (g,) = torch.autograd.grad(out, t, gout)
    n = i.numel()
    add = lambda y: torch.zeros(30, t[0].numel(), dtype=torch.float64, device=DEV).index_add_(  # noqa: E731
        0, i.reshape(-1), y.double().reshape(n, -1))
    uses = torch.bincount(i.reshape(-1), minlength=30)[:, None]
    assert g.shape == t.shape
    assert ((g.double().reshape(30, -1) - add(gout)).abs() <= (uses + 3) * U * add(gout.abs())).all()


@pytest.mark.parametrize("N", [500, 50000])
@pytest.mark.parametrize("C", [5, 64, 3001])
def test_one_gradient_alone(N, C):
    """Only the table, or only the weights, ask for a gradient: as when both do, up to the order in which the
    terms are added ((n + 3) u sum|f g| of a row's n uses and (C + 3) u sum|g t|, on each side)."""
    from tt_splat_b200 import binned
    x = _inputs(40, C, (N,), seed=C)
    _, (gt, gw) = _check(x)
    t = x["table"].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(binned.gather_rows(t, x["idx"], x["valid"], x["weight"]), t, x["gout"])
    use = (x["idx"] >= 0) & x["valid"]
    term = (x["weight"][use, None].double() * x["gout"][use].double()).abs()
    mag = torch.zeros(40, C, dtype=torch.float64, device=DEV).index_add_(0, x["idx"][use], term)
    uses = torch.bincount(x["idx"][use], minlength=40)[:, None]
    assert ((g.double() - gt.double()).abs() <= 2 * (uses + 3) * U * mag).all()
    w = x["weight"].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(binned.gather_rows(x["table"], x["idx"], x["valid"], w), w, x["gout"])
    tab = x["table"].double()[x["idx"].clamp(min=0)]
    assert ((g.double() - gw.double()).abs() <= 2 * (C + 3) * U * (tab * x["gout"].double()).abs().sum(1)).all()


def test_many_unused():
    """Nothing, or a single slot, of many looked up: every row is written all the same."""
    x = _inputs(70001, 3, (20000,), unused=0.0)
    x["valid"][:] = False
    _check(x)
    x["valid"][12345] = True
    _check(x)


@pytest.mark.parametrize("dt", TYPES)
def test_strided_tables_and_gradients(dt):
    """Columns of a wider table, an offset that breaks 16-byte alignment, and gradients that arrive as a
    slice or as one expanded row or number."""
    from tt_splat_b200 import binned
    wide = torch.randn(40, 24, device=DEV).to(dt)
    i = torch.randint(0, 40, (100,), device=DEV)
    for cols in (slice(0, 8), slice(1, 9), slice(2, 5), slice(8, 24)):
        assert torch.equal(binned.gather_rows(wide[:, cols], i), wide[i][:, cols])
    assert torch.equal(binned.gather_rows(wide.t(), i % 24), wide.t()[i % 24])
    x = _inputs(40, 8, (100,), dt)
    big = torch.randn(100, 19, device=DEV).to(dt)
    _check(x, gout=big[:, 3:11])
    _check(x, gout=big[:1, :8].expand(100, 8))
    _check(x, gout=big[:1, :1].expand(100, 8))
    x["table"] = wide[:, 5:13]
    _check(x)


def test_bad_values_stay_out():
    """NaN gradients and weights of unused slots, and table rows nobody uses, reach nothing; an index
    past the table gives NaN and no gradient."""
    from tt_splat_b200 import binned
    x = _inputs(20, 6, (200,), unused=0.0)
    x["valid"][::3] = False
    x["table"][7] = float("nan")
    x["idx"][x["idx"] == 7] = 8
    x["gout"][::3] = float("nan")
    y = dict(x, weight=x["weight"].clone())
    y["weight"][::3] = float("inf")
    t, w = y["table"].requires_grad_(True), y["weight"].requires_grad_(True)
    gt, gw = torch.autograd.grad(binned.gather_rows(t, y["idx"], y["valid"], w), [t, w], y["gout"])
    assert torch.isfinite(gt).all() and torch.isfinite(gw).all() and (gw[::3] == 0).all()
    assert torch.isfinite(binned.gather_rows(y["table"], y["idx"], y["valid"], y["weight"])).all()
    for far in (20, 21, 2 ** 31 - 1, 2 ** 40):
        t = torch.randn(20, 6, device=DEV, requires_grad=True)
        w = torch.ones(3, device=DEV, requires_grad=True)
        out = binned.gather_rows(t, torch.tensor([1, far, 1], device=DEV), weight=w)
        assert out[1].isnan().all() and torch.equal(out[0], t[1])
        gt, gw = torch.autograd.grad(out, [t, w], torch.ones_like(out))
        assert torch.equal(gt[1], torch.full((6,), 2.0, device=DEV)) and gt.sum() == 12 and gw[1] == 0


def test_offsets_past_32_bits():
    """An output and a table whose last elements lie past 2^31 elements."""
    from tt_splat_b200 import binned
    C = 8192
    R = 2 ** 31 // C + 3
    t = torch.zeros(R, C, dtype=torch.bfloat16, device=DEV)
    t[-1] = 1.5
    t[0] = 0.5
    i = torch.zeros(R, dtype=torch.int32, device=DEV)
    i[-1] = R - 1
    t.requires_grad_(True)
    out = binned.gather_rows(t, i)
    assert (out[-1] == 1.5).all() and (out[-2] == 0.5).all()
    gout = torch.zeros_like(out)
    gout[-1], gout[-2] = 2.0, 3.0
    (g,) = torch.autograd.grad(out, t, gout)
    assert (g[-1] == 2.0).all() and (g[0] == 3.0).all() and (g[1:-1] == 0).all()


def test_same_bits_every_time():
    a, b = (_check(_inputs(64, 40, (30000,), torch.bfloat16, hot=0.3)) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a[1], b[1]))


def test_gradient_against_differences():
    """The lookup is linear in the table and in the weights, so differences are exact up to rounding: the
    change of <gout, out> along a direction d equals <gradient, d> (fp32 sums of 4000 terms, 4000 u)."""
    from tt_splat_b200 import binned
    x = _inputs(30, 8, (500,))
    _, (gt, gw) = _check(x, scale=2.0)
    value = lambda t, w: (binned.gather_rows(t, x["idx"], x["valid"], w, 2.0).double() * x["gout"].double()).sum()  # noqa: E731
    d, e = torch.randn_like(x["table"]), torch.randn_like(x["weight"])
    dt = value(x["table"] + d, x["weight"]) - value(x["table"], x["weight"])
    dw = value(x["table"], x["weight"] + e) - value(x["table"], x["weight"])
    mag = (x["gout"].double().abs().sum() * 40)
    assert abs(dt - (gt.double() * d.double()).sum()) < 4000 * U * mag
    assert abs(dw - (gw.double() * e.double()).sum()) < 4000 * U * mag


def test_streams_and_graphs():
    """On a side stream, two calls at once on two streams, and a captured forward and backward replayed on
    new contents."""
    from tt_splat_b200 import binned
    x = _inputs(100, 33, (20000,), hot=0.2)
    y = _inputs(900, 4, (9000,), torch.float16, seed=5)
    ref = [_check(z) for z in (x, y)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for z, s in zip((x, y), streams):
        with torch.cuda.stream(s):
            t, w = z["table"].detach().requires_grad_(True), z["weight"].detach().requires_grad_(True)
            out = binned.gather_rows(t, z["idx"], z["valid"], w)
            got.append((out, torch.autograd.grad(out, [t, w], z["gout"])))
    torch.cuda.synchronize()
    for (o, g), (ro, rg) in zip(got, ref):
        assert torch.equal(o, ro) and all(torch.equal(a, b) for a, b in zip(g, rg))

    t, w = x["table"].clone().requires_grad_(True), x["weight"].clone().requires_grad_(True)
    # torch ties a leaf's gradient to the stream of the graph that is alive: eager ones go before the capture
    eager = binned.gather_rows(t, x["idx"], x["valid"], w)
    del eager
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = binned.gather_rows(t, x["idx"], x["valid"], w)
            grads = torch.autograd.grad(out, [t, w], x["gout"])
        graphs.append((g, out, grads))
    z = _inputs(100, 33, (20000,), seed=9, hot=0.1)
    with torch.no_grad():
        t.copy_(z["table"]), w.copy_(z["weight"])
        x["idx"].copy_(z["idx"]), x["valid"].copy_(z["valid"]), x["gout"].copy_(z["gout"])
    for g, _, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    ro, rg = _check(z)
    for _, o, gr in graphs:
        assert torch.equal(o, ro) and all(torch.equal(a, b) for a, b in zip(gr, rg))


def test_second_derivative_is_refused():
    from tt_splat_b200 import binned
    t = torch.randn(5, 3, device=DEV, requires_grad=True)
    out = binned.gather_rows(t, torch.zeros(4, dtype=torch.int64, device=DEV))
    (g,) = torch.autograd.grad((out * out).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), t)


def test_forward_mode_is_refused():
    """A tangent of an input or of an incoming gradient raises; plain tensors beside a dual level do not."""
    import torch.autograd.forward_ad as fw
    from tt_splat_b200 import binned
    t, w = torch.randn(6, 3, device=DEV, requires_grad=True), torch.rand(4, device=DEV)
    i = torch.tensor([1, 2, 5, 1], device=DEV)
    dual = lambda x: fw.make_dual(x.detach(), torch.ones_like(x))  # noqa: E731
    with fw.dual_level():
        for args in ((dual(t), i), (t, i, None, dual(w))):
            for grad in (False, True):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    binned.gather_rows(*args)
        out = binned.gather_rows(t, i, weight=w)
        assert torch.equal(out, w[:, None] * t[i])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, t, dual(out))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: binned.gather_rows(x, i), (t.detach(),), (torch.ones(6, 3, device=DEV),))


def test_negated_views():
    """Tensors that only say that their numbers are negated, as the imaginary part of a conjugate does: the same
    bits as their copies give, forward and backward (negation rounds nothing)."""
    from tt_splat_b200 import binned
    x = _inputs(40, 6, (300,), hot=0.2)
    neg = torch._neg_view
    _check(dict(x, table=neg(x["table"])))
    _check(dict(x, weight=neg(x["weight"])))
    _check(x, gout=neg(x["gout"]))
    out = binned.gather_rows(neg(x["table"]), x["idx"], x["valid"], neg(x["weight"]))
    assert torch.equal(out, binned.gather_rows(x["table"], x["idx"], x["valid"], x["weight"]))
    z = torch.complex(torch.randn(40, device=DEV), torch.randn(40, device=DEV))
    i = x["idx"].clamp(min=0)
    assert z.conj().imag.is_neg() and torch.equal(binned.gather_rows(z.conj().imag, i), -z.imag[i])
    t = x["table"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(binned.gather_rows(neg(t), i), t, x["gout"])
    (h,) = torch.autograd.grad(binned.gather_rows(t, i), t, x["gout"])
    assert torch.equal(g, -h)


@pytest.mark.parametrize("op", ["rows", "labels"])
def test_other_threads_go_on(op):
    """While calls wait for room in the GPU's queue, which a sleep of about a second blocks, a thread that wakes every
    millisecond never stands still for half of it."""
    import threading
    import time

    from tt_splat_b200 import binned, metrics
    t, i = torch.randn(100, 16, device=DEV), torch.randint(0, 16, (100,), device=DEV)
    call = (lambda: binned.gather_rows(t, i)) if op == "rows" else (lambda: metrics.label_log_probs(t, i))
    call()
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    stop, gaps = threading.Event(), [0.0]

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    thread = threading.Thread(target=tick)
    thread.start()
    start.record()
    torch.cuda._sleep(2_000_000_000)               # clock cycles
    end.record()
    n = 0
    while not end.query() and n < 20000:
        call()
        n += 1
    stop.set()
    thread.join()
    torch.cuda.synchronize()
    assert max(gaps) < 0.5e-3 * start.elapsed_time(end)


def test_saved_tensors_through_python_hooks():
    """Hooks that pack what the functions save, which run Python inside the calls: the same bits."""
    from tt_splat_b200 import binned, metrics
    x = _inputs(40, 6, (300,))
    y, lab = torch.randn(30, 9, device=DEV), torch.randint(0, 9, (30,), device=DEV)
    packed = []

    def both():
        t, w = x["table"].clone().requires_grad_(True), x["weight"].clone().requires_grad_(True)
        rows = torch.autograd.grad(binned.gather_rows(t, x["idx"], x["valid"], w), [t, w], x["gout"])
        leaf = y.clone().requires_grad_(True)
        s = metrics.label_log_probs(leaf, lab, top=2)
        return *rows, *torch.autograd.grad(s.logp.sum() + s.entropy.sum(), leaf)

    want = both()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(0) or t.cpu(), lambda t: t.to(DEV)):
        got = both()
    assert len(packed) >= 5 and all(torch.equal(a, b) for a, b in zip(got, want))


# Sums of small whole numbers (and halves) are exact in fp32 whatever their order, as long as they stay below
# 2^24 steps: a lost or doubled term of a row with many uses shows, which a bound that grows with the uses hides.
def _check_whole(rows, N, C, dt, weight, seed=0, unused=0):
    """A table gradient (and the weights') whose uses are `rows` in a random order, N of them after padding with
    unused slots, against the integers."""
    from tt_splat_b200 import binned
    g = torch.Generator(device=DEV).manual_seed(seed)
    idx = torch.cat([rows, torch.full((N - rows.numel(),), -1, device=DEV)])[torch.randperm(N, generator=g, device=DEV)]
    R = int(rows.max()) + 2
    gout = torch.randint(-3, 4, (N, C), generator=g, device=DEV)
    gout[:, 0] = 1                                            # counts the uses
    table = torch.randint(-2, 3, (R, C), generator=g, device=DEV).to(dt).requires_grad_(True)
    twice = torch.randint(1, 5, (N,), generator=g, device=DEV)      # weights of 0.5, 1, 1.5 and 2
    w = (twice.float() * 0.5).requires_grad_(True) if weight else None
    out = binned.gather_rows(table, idx, weight=w)
    grads = torch.autograd.grad(out, [table] + ([w] if weight else []), gout.to(dt))
    f = twice if weight else torch.full_like(twice, 2)
    n = idx >= 0
    ref = torch.zeros(R, C, dtype=torch.float64, device=DEV).index_add_(0, idx[n], (f[n, None] * gout[n]).double())
    assert ref.abs().max() < 2 ** 24
    assert torch.equal(grads[0], (ref * 0.5).to(dt))
    if weight:
        dots = (gout * table.detach().long()[idx.clamp(min=0)]).sum(1)
        assert torch.equal(grads[1], torch.where(n, dots, 0).float())


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("dt,C", [(torch.float32, 1), (torch.float32, 6), (torch.float32, 45), (torch.bfloat16, 64),
                                  (torch.float32, 128), (torch.float16, 45), (torch.float32, 300)])
@pytest.mark.parametrize("N", [9000, 70001, 300000])
def test_hot_rows_exactly(N, dt, C, weight):
    """One row with nearly all uses, first, in the middle and last among the rows, and a few hot rows in turn."""
    for hot, share in ((0, 0.9), (500, 0.81), (999, 0.99), (3, 1.0)):
        n = int(N * share)
        others = torch.randint(0, 1000, (N - n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(hot))
        _check_whole(torch.cat([torch.full((n,), hot, device=DEV), others]), N + 17, C, dt, weight, seed=hot)
    _check_whole(torch.arange(N, device=DEV) % 5 * 7, N, C, dt, weight)


@pytest.mark.parametrize("N,C", [(9000, 128), (60000, 32), (60000, 128), (300000, 64), (300000, 128)])
def test_rows_on_the_borders_of_chunks(N, C):
    """All rows have the same number of uses: every whole multiple of 8 up to 128, which the chunks' lengths are, so
    that rows begin and end where chunks do, and one more and less; 2 to 4 of them, where a row is first split, and
    31 to 35, where its parts are joined in another way."""
    for L in range(8, 129, 8):
        for m in (1, 2, 3, 4, 31, 32, 33, 34, 35):
            for d in (-1, 0, 1):
                size = L * m + d
                k = N // size
                if k and (d == 0 or m in (2, 33)):
                    _check_whole(torch.arange(k, device=DEV).repeat_interleave(size), k * size, C, torch.float32, (L + m) % 2 == 0, seed=L)


def test_gradients_not_asked_for_are_not_computed():
    """Where both inputs require gradients and one is asked for, the other one takes no memory, and the one that is
    asked for has the bits of the same call with the other input constant."""
    from tt_splat_b200 import binned
    x = _inputs(1000000, 16, (3000,), unused=0.1)
    t, w = x["table"].requires_grad_(True), x["weight"].requires_grad_(True)

    def one(table, weight, of):
        out = binned.gather_rows(table, x["idx"], x["valid"], weight)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        (g,) = torch.autograd.grad(out, of, x["gout"])
        return g, torch.cuda.max_memory_allocated() - before

    g, peak = one(t, w, w)
    assert torch.equal(g, one(t.detach(), w, w)[0]) and peak < t.numel()
    assert torch.equal(one(t, w, t)[0], one(t, w.detach(), t)[0])
    leaf = torch.zeros((), device=DEV, requires_grad=True)          # inputs that are no leaves themselves
    out = binned.gather_rows(t + leaf, x["idx"], x["valid"], w * 1)
    (h,) = torch.autograd.grad(out, w, x["gout"])
    assert torch.equal(h, g)
    out = binned.gather_rows(t, x["idx"], x["valid"])
    assert torch.autograd.grad(out, t, x["gout"])[0].shape == t.shape
    t.grad = w.grad = None
    binned.gather_rows(t, x["idx"], x["valid"], w).backward(x["gout"])      # everything
    both = torch.autograd.grad(binned.gather_rows(t, x["idx"], x["valid"], w), [t, w], x["gout"])
    assert torch.equal(t.grad, both[0]) and torch.equal(w.grad, both[1])
