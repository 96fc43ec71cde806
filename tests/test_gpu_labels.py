"""Label log probabilities, entropies and alternatives (metrics.label_log_probs) and their gradient
against float64, at the sizes and masks where they can go wrong.

Tolerances, with u = 2^-24: d = x - m is off by u |d|; exp of it, computed as 2^(d log2 e), by |d| u for
the product, 2^-22 = 4u for the power and u |d| for d, together (2|d| + 4) u relative, so the sum S by
e_S = u (2 D + 4 + n) with D = sum p |d| and n additions on the longest path of a sum: ceil(C / 32) + 16
where a warp or a block shares a row; C / 4 + 6 where one thread takes a row of up to 256 labels in four
sums (up to 3 labels more in one, and 3 additions of the sums).  From there:
* log S: e_S + 4u (1 + log S);  log p_j: u |d_j| + that + u |log p_j|;
* A / S with A = sum e d: u sum p |d| (2|d| + 5 + n) + e_S D, and H adds the error of log S and u H;
* p_j: relative, the error of log p_j + (|log p_j| + 4) u;
* dx_j: the errors of p_j and log p_j + H times their factors, 6u of the terms' magnitudes (a sum of up to
  top + 3 terms adds u each), and the rounding of the result, finfo(type).eps / 2.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(P, C, dt=torch.float32, seed=0, masked=0.0, unlabelled=0.1, spread=3.0, index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(P, C, generator=g) * spread
    x[torch.rand(P, C, generator=g) < masked] = -math.inf
    t = torch.randint(0, C, (P,), generator=g)
    t[torch.rand(P, generator=g) < unlabelled] = -1
    return x.to(dt).to(DEV), t.to(index).to(DEV)


def _reference(x, t, top):
    x = x.double()
    P, C = x.shape
    some = (x > -math.inf).any(1)
    # m first, then log S: beside a maximum of -3.4e38 (a row of fp32 lowest values) one step of a float64
    # is 2^75, and m + log S would lose log S
    m = torch.where(some, x.max(1).values, 0.0)
    logS = torch.where(some, (x - m[:, None]).exp().sum(1).log(), 0.0)
    lp = (x - m[:, None]) - logS[:, None]
    p = lp.exp()
    H = -torch.special.xlogy(p, p).sum(1)
    H = torch.where(some, H, 0.0)
    logp = torch.where(t >= 0, lp.gather(1, t.clamp(min=0).long()[:, None])[:, 0], 0.0)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(top, C)
    ids = torch.full((P, top), -1, dtype=torch.int64, device=DEV)
    tlp = torch.full((P, top), -math.inf, dtype=torch.float64, device=DEV)
    ids[:, :k] = torch.where(v[:, :k] > -math.inf, i[:, :k], -1)
    tlp[:, :k] = torch.where(v[:, :k] > -math.inf, (v[:, :k] - m[:, None]) - logS[:, None], -math.inf)
    # error bounds of the header
    d = torch.where(p > 0, (x - m[:, None]).abs(), 0.0)
    n = max((C + 31) // 32 + 16, C // 4 + 6 if C <= 256 else 0)
    D, D2 = (p * d).sum(1), (p * d * d).sum(1)
    eS = U * (2 * D + 4 + n)
    eL = eS + 4 * U * (1 + logS)
    eH = U * (2 * D2 + (5 + n) * D) + eS * D + eL + U * H.abs() + 4 * U * D
    flp = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
    # far below the maximum d is large whatever p
    dd = torch.where(torch.isfinite(x), (x - m[:, None]).abs(), 0.0)
    elp = U * dd + eL[:, None] + U * flp
    return dict(lp=lp, p=p, H=H, logp=logp, ids=ids, tlp=tlp, some=some, eH=eH, elp=elp, flp=flp)


def _close(got, ref, tol):
    same = got.double() == ref                                # infinities
    return (same | ((got.double() - ref).abs() <= tol * 1.01)).all()


def _check(x, t, top=0, grads=("logp", "entropy", "top"), seed=1):
    from tt_splat_b200 import metrics
    leaf = x.detach().requires_grad_(True)
    s = metrics.label_log_probs(leaf, t, top=top)
    P, C, dt = x.shape[0], x.shape[1], x.dtype
    R = _reference(x, t, top)
    tl = t.long()
    et = R["elp"].gather(1, tl.clamp(min=0)[:, None])[:, 0]
    assert s.logp.shape == (P,) and s.logp.dtype == torch.float32
    assert _close(s.logp.detach(), R["logp"], et)
    assert _close(s.entropy.detach(), R["H"], R["eH"])
    assert s.top_ids.dtype == torch.int64 and torch.equal(s.top_ids, R["ids"])
    if top:
        ek = R["elp"].gather(1, R["ids"].clamp(min=0))
        assert _close(s.top_logp.detach(), R["tlp"], ek)
    g = torch.Generator().manual_seed(seed)
    gl = torch.randn(P, generator=g).to(DEV) if "logp" in grads else None
    gh = torch.randn(P, generator=g).to(DEV) if "entropy" in grads else None
    gt = torch.randn(P, top, generator=g).to(DEV) if "top" in grads and top else None
    outs = [(o, q) for o, q in ((s.logp, gl), (s.entropy, gh), (s.top_logp, gt)) if q is not None]
    (gx,) = torch.autograd.grad([o for o, _ in outs], leaf, [q for _, q in outs])
    z = torch.zeros(P, dtype=torch.float64, device=DEV)
    gl = z if gl is None else torch.where(tl >= 0, gl.double(), z)
    gh = z if gh is None else gh.double()
    up = torch.zeros(P, C, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(up)
    up.scatter_add_(1, tl.clamp(min=0)[:, None], gl[:, None])
    mag.scatter_add_(1, tl.clamp(min=0)[:, None], gl.abs()[:, None])
    if gt is not None:
        k = torch.where(R["ids"] >= 0, gt.double(), 0.0)
        up.scatter_add_(1, R["ids"].clamp(min=0), k)
        mag.scatter_add_(1, R["ids"].clamp(min=0), k.abs())
    total, tmag = up.sum(1, keepdim=True), mag.sum(1, keepdim=True)
    p, live = R["p"], R["p"] > 0
    lpH = torch.where(live, R["lp"] + R["H"][:, None], 0.0)
    ref = up - p * total - gh[:, None] * p * lpH
    ref = torch.where(R["some"][:, None], ref, 0.0)
    ep = R["elp"] + (R["flp"] + 4) * U
    body = p * (tmag + gh.abs()[:, None] * lpH.abs())
    tol = body * (ep + (top + 6) * U) + p * gh.abs()[:, None] * (R["elp"] + R["eH"][:, None]) + (top + 3) * U * mag
    r = torch.finfo(dt).eps / 2
    tol = tol * (1 + r) + ref.abs() * r + (2.0 ** -25 if dt == torch.float16 else 1e-37)
    assert gx.shape == x.shape and gx.dtype == dt and _close(gx, ref, tol)
    return s, gx


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", [1, 2, 3, 7, 8, 16, 21, 32, 33, 64, 100, 128, 150, 255, 256, 257, 600, 1000, 1024, 2047, 4097,
                               8192, 20001, 70000])
def test_label_counts(C, dt):
    x, t = _inputs(37, C, dt, seed=C)
    _check(x, t, top=5)


@pytest.mark.parametrize("P", [1, 2, 5, 31, 33, 127, 129, 1000, 4099])
@pytest.mark.parametrize("C", [5, 64, 333])
def test_row_counts(P, C):
    x, t = _inputs(P, C, seed=P, index=torch.int32)
    _check(x, t, top=3)


@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 16, 21, 33, 64, 100, 127, 128, 150, 200, 255, 256, 257])
def test_many_rows_of_few_labels(C):
    """As many rows as an image has: odd and even row sizes on both sides of what a thread's tile takes, a
    last tile that is not full, ties and masks among them."""
    for k, dt in enumerate(TYPES):
        x, t = _inputs(38007, C, dt, seed=C, masked=0.2, index=torch.int32 if k else torch.int64)
        x[::3] = (x[::3] * 0.5).round()
        x[1::997] = -math.inf
        x[2::997] = 1.0
        _check(x, t, top=(3, 7, 0)[(C + k) % 3], grads=("logp", "entropy", "top") if (C + k) % 3 < 2 else ("logp",))
        if C in (21, 64, 150):
            for top in (1, 2, 4, 16):
                _check(x, t, top=top, grads=("logp",))


@pytest.mark.parametrize("P,C", [(1801, 1025), (1776, 1500), (2000, 2048), (1900, 4095), (1777, 4096), (1800, 4097)])
def test_many_rows_of_some_thousand_labels(P, C):
    """Both sides of what a warp takes for itself, with ties, masks, bad and empty rows, and rows that start at
    every offset from a 16-byte boundary, their gradients' offset another one too."""
    from tt_splat_b200 import metrics
    for k, dt in enumerate(TYPES):
        x, t = _inputs(P, C, dt, seed=C + k, masked=0.3 * k)
        x[::3] = (x[::3] * 0.5).round()
        x[1::97] = -math.inf
        x[2::97] = 1.0
        x[4::97, C // 2:] = 9.0
        x[5::97] = torch.finfo(dt).min
        _check(x, t, top=(8, 16, 1)[k])
        wide = torch.randn(P, C + 5, device=DEV).to(dt)
        wide[:, 1:-4] = x
        leaf = wide[:, 1:-4].detach().requires_grad_(True)
        s, q = metrics.label_log_probs(leaf, t, top=3), metrics.label_log_probs(x, t, top=3)
        tol = 2 * _reference(x, t, 0)["elp"].gather(1, t.clamp(min=0)[:, None])[:, 0]
        assert torch.equal(s.top_ids, q.top_ids) and _close(s.logp.detach(), q.logp.double(), tol)
        (g,) = torch.autograd.grad(s.logp, leaf, torch.ones(P, device=DEV))
        y = x.detach().requires_grad_(True)
        (h,) = torch.autograd.grad(metrics.label_log_probs(y, t).logp, y, torch.ones(P, device=DEV))
        # each is within its bound of the exact one, at most (5 |log p| + n + 30) u of p on each side, and rounded
        p = _reference(x, t, 0)["p"]
        far = (p * (5 * 80 + C / 32 + 60) * 2 * U + 2 * torch.finfo(dt).eps / 2 * h.double().abs() + 2.0 ** -24)
        assert ((g.double() - h.double()).abs() <= far).all()
        z = x.clone()
        z[7, C - 1], z[8, 0], z[9, 5] = math.nan, math.inf, math.nan
        t[7], t[8], t[9], t[11] = 0, 0, -1, C
        s = metrics.label_log_probs(z.requires_grad_(True), t, top=2)
        (g,) = torch.autograd.grad(s.logp, z, torch.ones(P, device=DEV))
        assert s.logp[7:9].isnan().all() and s.logp[9] == 0 and s.logp[11].isnan() and s.entropy[7:10].isnan().all()
        assert (s.top_ids[7:10] == -1).all() and g[7:9].isnan().all() and (g[9] == 0).all() and g[11].isnan().all()


def test_many_rows_bad_values():
    from tt_splat_b200 import metrics
    x, t = _inputs(40000, 20, unlabelled=0.0)
    x[7, 3], x[8, 0], x[9, 19] = math.nan, math.inf, math.nan
    t[9], t[10] = -1, 20
    leaf = x.requires_grad_(True)
    for top in (2, 6):
        s = metrics.label_log_probs(leaf, t, top=top)
        (g,) = torch.autograd.grad(s.logp, leaf, torch.ones(40000, device=DEV))
        bad = torch.zeros(40000, dtype=torch.bool, device=DEV)
        bad[7], bad[8], bad[10] = True, True, True
        assert torch.equal(s.logp.isnan(), bad) and s.logp[9] == 0
        assert torch.equal(g.isnan().all(1), bad) and torch.equal(g.isnan().any(1), bad) and (g[9] == 0).all()
        assert (s.top_ids[7:10] == -1).all() and s.top_logp[7:10].isnan().all() and (s.top_ids[10:] >= 0).all()


@pytest.mark.parametrize("P,C", [(1, 131072), (2, 65537), (5, 32000), (148, 16384), (300, 50257), (700, 9001)])
def test_few_rows_many_labels(P, C):
    for dt in TYPES:
        x, t = _inputs(P, C, dt, seed=P)
        _check(x, t, top=16)


@pytest.mark.parametrize("top", [0, 1, 2, 8, 15, 16])
@pytest.mark.parametrize("C", [4, 16, 40, 1500, 40000])
def test_tops(top, C):
    x, t = _inputs(9, C, torch.float16, seed=top)
    _check(x, t, top=top)


@pytest.mark.parametrize("C", [3, 16, 50, 200, 1030, 5000, 40000])
def test_ties(C):
    """Few distinct values, all equal, and a run of the largest value: the lowest ids win."""
    for dt in TYPES:
        x, t = _inputs(13, C, dt, spread=1.0)
        x = (x * 1.5).round()
        x[0] = 2.0
        x[1] = -0.0
        x[1, ::2] = 0.0
        x[2, C // 2:] = 9.0
        x[3] = torch.arange(C, device=DEV).to(dt) / C
        x[4] = -torch.arange(C, device=DEV).to(dt) / C
        _check(x, t, top=16)


@pytest.mark.parametrize("C", [2, 21, 150, 1000, 9000, 40000])
def test_masks(C):
    for dt in TYPES:
        x, t = _inputs(40, C, dt, seed=C, masked=0.7)
        x[0] = -math.inf                      # nothing left, labelled and not
        x[1] = -math.inf
        t[0], t[1] = 0, -1
        x[2] = -math.inf
        x[2, C - 1] = 1.0                     # one label left, the given one masked
        t[2] = 0
        x[3] = -math.inf
        x[3, C // 2] = -5.0
        t[3] = C // 2
        x[4] = torch.finfo(dt).min            # masks of the type's lowest value
        x[5] = torch.finfo(dt).min
        x[5, 0] = 3.0
        s, gx = _check(x, t, top=4)
        assert s.logp[0] == -math.inf and s.logp[1] == 0 and s.entropy[0] == 0
        assert (s.top_ids[:2] == -1).all() and (gx[:2] == 0).all()
        assert s.top_ids[2].tolist() == [C - 1, -1, -1, -1] and s.logp[2] == -math.inf
        assert s.logp[3] == 0 and s.entropy[3] == 0


@pytest.mark.parametrize("C", [5, 150, 3001, 40000])
def test_nan_infinite_and_bad_labels(C):
    from tt_splat_b200 import metrics
    x, t = _inputs(8, C, unlabelled=0.0)
    x[0, C // 2] = math.nan
    x[1, 0] = math.inf
    x[2, C - 1] = math.nan
    x[3, 0] = math.nan
    t[2] = t[3] = -1
    t[5], t[6], t[7] = C, 2 ** 31 - 1, 2 ** 40
    leaf = x.requires_grad_(True)
    s = metrics.label_log_probs(leaf, t, top=2)
    assert s.logp[:2].isnan().all() and (s.logp[2:4] == 0).all() and torch.isfinite(s.logp[4]) and s.logp[5:].isnan().all()
    assert s.entropy[:4].isnan().all() and torch.isfinite(s.entropy[4:]).all()
    assert (s.top_ids[:4] == -1).all() and s.top_logp[:4].isnan().all() and (s.top_ids[4:] >= 0).all()
    gl = torch.ones(8, device=DEV)
    (g,) = torch.autograd.grad(s.logp, leaf, gl, retain_graph=True)
    assert g[:2].isnan().all() and (g[2:4] == 0).all() and torch.isfinite(g[4]).all() and g[5:].isnan().all()
    gl[:] = 0
    (g,) = torch.autograd.grad(s.logp, leaf, gl)
    assert (g[:5] == 0).all()


@pytest.mark.parametrize("P,C", [(8, 5), (8, 150), (8, 3001), (40000, 21)])
def test_bad_labels_left_out_of_the_loss(P, C):
    """A label past the last whose log probability does not reach the loss leaves its row's gradient zero."""
    from tt_splat_b200 import metrics
    x, t = _inputs(P, C, seed=3, unlabelled=0.0)
    t[2], t[5] = C, 2 ** 31 - 1
    leaf = x.requires_grad_(True)
    s = metrics.label_log_probs(leaf, t)
    (g,) = torch.autograd.grad(torch.where(t < C, s.logp, 0.0).sum(), leaf)
    assert (g[2] == 0).all() and (g[5] == 0).all() and torch.isfinite(g).all() and (g[:2] != 0).any(1).all()


@pytest.mark.parametrize("grads", [("logp",), ("entropy",), ("top",), ("logp", "top")])
@pytest.mark.parametrize("C", [11, 300, 12000])
def test_each_gradient_alone(grads, C):
    x, t = _inputs(30, C, seed=4)
    _check(x, t, top=3, grads=grads)


@pytest.mark.parametrize("C", [7, 500])
def test_gradient_against_differences(C):
    """Central differences of the operator's own outputs, summed in float64: step h = 2^-6 leaves
    h^2 / 6 of a third derivative (below 2 for a log probability and below 4 log C for the entropy,
    times the squared step's own size) and 2 (C u + 2^-20) / 2h of rounding."""
    from tt_splat_b200 import metrics
    x, t = _inputs(4, C, seed=8, unlabelled=0.0, spread=1.0)
    _, _ = _check(x, t)
    leaf = x.clone().requires_grad_(True)
    s = metrics.label_log_probs(leaf, t)
    (g,) = torch.autograd.grad([s.logp, s.entropy], leaf, [torch.ones(4, device=DEV), torch.full((4,), 0.5, device=DEV)])
    h = 2.0 ** -6
    val = lambda y: (lambda s: s.logp.double() + 0.5 * s.entropy.double())(metrics.label_log_probs(y, t))  # noqa: E731
    for j in range(0, C, max(1, C // 7)):
        e = torch.zeros_like(x)
        e[:, j] = h
        fd = (val(x + e) - val(x - e)) / (2 * h)
        assert ((fd - g[:, j].double()).abs() < h * h / 6 * (2 + 4 * math.log(C)) + (C * U + 2.0 ** -20) / h).all()


def test_large_logits():
    """Logits of a few thousands: differences decide, not sizes."""
    x, t = _inputs(20, 900, seed=6)
    _check(x + 4000.0, t, top=3)
    _check(x * 300.0, t, top=3)


@pytest.mark.parametrize("dt", TYPES)
def test_layouts(dt):
    """Leading dimensions, slices of wider rows (aligned or not), expanded rows and transposed logits."""
    from tt_splat_b200 import metrics
    img = torch.randn(6, 10, 40, device=DEV).to(dt)
    lab = torch.randint(-1, 13, (6, 10), device=DEV)
    for cols in (slice(0, 13), slice(1, 14), slice(8, 21)):
        y = img[..., cols]
        leaf = y.detach().requires_grad_(True)
        s = metrics.label_log_probs(leaf, lab, top=2)
        flat, gx = _check(y.contiguous().reshape(60, 13), lab.reshape(60), top=2, grads=("logp",))
        assert s.logp.shape == (6, 10) and s.top_ids.shape == (6, 10, 2)
        # another layout may add in another order: each result is within its bound of the exact one
        R = _reference(y.reshape(60, 13), lab.reshape(60), 2)
        tol = 2 * R["elp"].gather(1, lab.reshape(60).clamp(min=0)[:, None])[:, 0]
        assert _close(s.logp.detach().reshape(-1), flat.logp.detach().double(), tol)
        assert torch.equal(s.top_ids.reshape(60, 2), flat.top_ids)
        two = y[0].detach().requires_grad_(True)
        s2 = metrics.label_log_probs(two, lab[0])
        (g2,) = torch.autograd.grad(s2.logp.sum(), two)
        assert _close(s2.logp.detach(), flat.logp[:10].detach().double(), tol[:10]) and g2.shape == two.shape
    one = img[0, 0, :13]
    s = metrics.label_log_probs(one, lab[0, 0])
    assert s.logp.shape == ()
    e = metrics.label_log_probs(one.expand(7, 13), torch.arange(7, device=DEV))
    x7 = one[None].repeat(7, 1)
    tol = 2 * _reference(x7, torch.arange(7, device=DEV), 0)["elp"][torch.arange(7), torch.arange(7)]
    assert _close(e.logp, metrics.label_log_probs(x7, torch.arange(7, device=DEV)).logp.double(), tol)
    tr = img[0, :, :].t()[:13]
    s = metrics.label_log_probs(tr, torch.zeros(13, dtype=torch.int64, device=DEV), top=1)
    assert torch.equal(s.logp, metrics.label_log_probs(tr.contiguous(), torch.zeros(13, dtype=torch.int64, device=DEV)).logp)
    none = metrics.label_log_probs(torch.empty(0, 5, device=DEV, dtype=dt), torch.empty(0, dtype=torch.int64, device=DEV), top=2)
    assert none.logp.shape == (0,) and none.top_ids.shape == (0, 2)


def test_offsets_past_32_bits():
    from tt_splat_b200 import metrics
    C = 65536
    P = 2 ** 31 // C + 2
    x = torch.zeros(P, C, dtype=torch.float16, device=DEV)
    x[-1, 5] = 8.0
    t = torch.full((P,), 5, dtype=torch.int64, device=DEV)
    x.requires_grad_(True)
    s = metrics.label_log_probs(x, t, top=2)
    want = 8.0 - math.log(math.exp(8.0) + C - 1)
    assert abs(s.logp[-1].item() - want) < 1e-4 and abs(s.logp[-2].item() + math.log(C)) < 1e-4
    assert s.top_ids[-1].tolist() == [5, 0] and s.top_ids[-2].tolist() == [0, 1]
    (g,) = torch.autograd.grad(s.logp, x, torch.ones(P, device=DEV))
    assert abs(g[-1, 5].item() - (1 - math.exp(want))) < 1e-3 and abs(g[-2, 5].item() - 1) < 1e-3


@pytest.mark.parametrize("P,C", [(5000, 21), (300, 1000), (2, 100000)])
def test_streams_and_graphs(P, C):
    from tt_splat_b200 import metrics
    x, t = _inputs(P, C, torch.bfloat16)
    y, v = _inputs(P, C, torch.bfloat16, seed=3)
    rx, ry = _check(x, t, top=3, grads=("logp",)), _check(y, v, top=3, grads=("logp",))
    gl = torch.randn(P, generator=torch.Generator().manual_seed(1)).to(DEV)
    torch.cuda.synchronize()
    got = []
    for (a, b) in ((x, t), (y, v)):
        with torch.cuda.stream(torch.cuda.Stream()):
            leaf = a.detach().requires_grad_(True)
            s = metrics.label_log_probs(leaf, b, top=3)
            got.append((s, torch.autograd.grad(s.logp, leaf, gl)[0]))
    torch.cuda.synchronize()
    for (s, g), (rs, rg) in zip(got, (rx, ry)):
        assert all(torch.equal(p, q) for p, q in zip(s, rs)) and torch.equal(g, rg)
    leaf, lab = x.clone().requires_grad_(True), t.clone()
    eager = metrics.label_log_probs(leaf, lab)
    del eager                                  # torch ties a leaf's gradient to the stream of a live graph
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = metrics.label_log_probs(leaf, lab, top=3)
            (gx,) = torch.autograd.grad(s.logp, leaf, gl)
        graphs.append((g, s, gx))
    with torch.no_grad():
        leaf.copy_(y), lab.copy_(v)
    for g, _, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, s, gx in graphs:
        assert all(torch.equal(p, q) for p, q in zip(s, ry[0])) and torch.equal(gx, ry[1])


def test_second_derivative_is_refused():
    from tt_splat_b200 import metrics
    x = torch.randn(5, 3, device=DEV, requires_grad=True)
    s = metrics.label_log_probs(x, torch.zeros(5, dtype=torch.int64, device=DEV))
    (g,) = torch.autograd.grad(s.logp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_rendered_labels_train_the_rows():
    """The whole path: label logits of a gaussian gathered through a view's tables, blended per pixel with
    the render's own weights, scored against a label image, and differentiated back to the table.  Against
    the same chain in float64 from the same weights.  The fp32 chain adds K = 128 products per pixel and
    label, each logit is off by (128 + 4) u times its magnitude, which the scores' derivative (at most 2)
    passes on; a row's gradient adds at most a few thousand such terms."""
    from tt_splat_b200 import binned, camera, metrics, model, synthetic
    sc = synthetic.config0(seed=0, G=600, res=64)
    m = model.GaussianModel.from_arrays(sc["params"], device=torch.device(DEV))
    cam = camera.Camera.from_dict(sc["cams"][0])
    tmap = binned.TileMap(64, 64)
    th, _, oc, w_b, (idx, valid) = binned._operands(m, cam, tmap, 1, 128)
    th, oc, w_b = th.detach(), oc.detach(), w_b.detach()
    C, T = 9, tmap.T
    g = torch.Generator().manual_seed(2)
    table = torch.randn(600, C, generator=g).to(DEV).requires_grad_(True)
    labels = torch.randint(-1, C, (64, 64), generator=g).to(DEV)
    w = torch.relu(torch.einsum("pc,tck->tpk", tmap.Phi, th)) ** 2 * oc.transpose(1, 2)
    w = w / (w.sum(2, keepdim=True) + w_b)

    def loss(rows, w, scores):
        logits = torch.empty(64 * 64, C, dtype=rows.dtype, device=DEV)
        logits = logits.index_copy(0, tmap.gidx, torch.einsum("tpk,tkc->tpc", w, rows).reshape(T * 256, C))
        lp, H = scores(logits.reshape(64, 64, C))
        return -lp.sum() / 4096 + 0.01 * H.sum() / 4096, logits

    def ours(x):
        s = metrics.label_log_probs(x, labels, top=3)
        return s.logp, s.entropy

    def plain(x):
        lp = torch.log_softmax(x, -1)
        one = lp.gather(-1, labels.clamp(min=0)[..., None])[..., 0]
        return torch.where(labels >= 0, one, 0.0), -(lp.exp() * lp).sum(-1)

    torch.backends.cuda.matmul.allow_tf32 = False
    got, logits = loss(binned.gather_rows(table, idx, valid), w, ours)
    (grad,) = torch.autograd.grad(got, table)
    t64 = table.detach().double().requires_grad_(True)
    ref, l64 = loss(t64[idx] * valid[..., None], w.double(), plain)
    (gref,) = torch.autograd.grad(ref, t64)
    e = (128 + 4) * U * table.detach().abs().max().item()
    assert (logits.double() - l64).abs().max() <= e
    assert abs(got.item() - ref.item()) <= 2 * (e + 64 * U * 10)
    # d loss / d row = sum over its (pixel, slot) uses of w_n d loss / d logit / 4096, |d| <= 1.2
    uses = torch.zeros(600, dtype=torch.float64, device=DEV).index_add_(0, idx[valid], w.double().sum(1)[valid])
    tol = uses / 4096 * (2 * e + 1.2 * (256 + 64 + 128) * U)
    assert ((grad.double() - gref).abs() <= tol[:, None] + 1e-12).all()
    assert gref.abs().max() > 100 * tol.max()


def test_forward_mode_is_refused():
    """A tangent of the logits or of an incoming gradient raises; plain tensors beside a dual level do not."""
    import torch.autograd.forward_ad as fw
    from tt_splat_b200 import metrics
    x, t = torch.randn(6, 3, device=DEV, requires_grad=True), torch.zeros(6, dtype=torch.int64, device=DEV)
    dual = lambda y: fw.make_dual(y.detach(), torch.ones_like(y))  # noqa: E731
    with fw.dual_level():
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                metrics.label_log_probs(dual(x), t)
        s = metrics.label_log_probs(x, t, top=2)
        for out in (s.logp, s.entropy, s.top_logp):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, x, dual(out), retain_graph=True)
        assert torch.isfinite(torch.autograd.grad(s.logp.sum(), x)[0]).all()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda y: metrics.label_log_probs(y, t).logp, (x.detach(),), (torch.ones(6, 3, device=DEV),))


def test_negated_views():
    """Tensors that only say that their numbers are negated, as the imaginary part of a conjugate does: the same
    bits as their copies give, forward and backward (negation rounds nothing)."""
    from tt_splat_b200 import metrics
    neg = torch._neg_view
    for C in (5, 700):
        x, t = _inputs(30, C, seed=C)
        _check(neg(x), t, top=3)
        s, gx = _check(x, t, top=3)
        leaf = x.clone().requires_grad_(True)
        g = [torch.randn(30, device=DEV), torch.randn(30, device=DEV), torch.randn(30, 3, device=DEV)]
        s = metrics.label_log_probs(leaf, t, top=3)
        outs = [s.logp, s.entropy, s.top_logp]
        (a,) = torch.autograd.grad(outs, leaf, [neg(q) for q in g], retain_graph=True)
        (b,) = torch.autograd.grad(outs, leaf, [-q for q in g])
        assert torch.equal(a, b)
        y = metrics.label_log_probs(neg(leaf), t, top=3)
        w = metrics.label_log_probs(-leaf.detach(), t, top=3)
        assert all(torch.equal(p, q) for p, q in zip(y, w))


@pytest.mark.parametrize("P,C", [(8, 5), (40000, 21), (8, 150), (40000, 300), (8, 1000), (1900, 3001), (8, 20001), (1300, 9001)])
def test_bad_rows_reached_by_the_alternatives_alone(P, C):
    """A row with NaN or +inf has NaN in the place of its alternatives' log probabilities: any gradient that is not
    zero makes its row NaN, gradients that cancel among them, and zeros leave it zero.  Its neighbours' rows are
    as they were without it."""
    from tt_splat_b200 import metrics
    for dt in TYPES:
        x, t = _inputs(P, C, dt, seed=C)
        t[1] = t[2] = t[4] = -1
        g = torch.randn(P, 3, generator=torch.Generator().manual_seed(3)).to(DEV)
        leaf = x.clone().requires_grad_(True)
        (clean,) = torch.autograd.grad(metrics.label_log_probs(leaf, t, top=3).top_logp, leaf, g)
        x[1, C // 2], x[2, 0], x[3, C - 1], x[4, 1], x[5] = math.nan, math.inf, math.nan, math.inf, -math.inf
        g[1] = torch.tensor([0.0, 0.0, 1.0])
        g[2] = torch.tensor([2.0, -2.0, 0.0])
        g[3:5] = 0.0
        leaf = x.requires_grad_(True)
        s = metrics.label_log_probs(leaf, t, top=3)
        assert s.top_logp[1:5].isnan().all() and (s.top_ids[1:6] == -1).all()
        (gx,) = torch.autograd.grad(s.top_logp, leaf, g)
        assert gx[1:3].isnan().all() and (gx[3:6] == 0).all()
        assert torch.equal(gx[6:], clean[6:]) and torch.equal(gx[0], clean[0])


@pytest.mark.parametrize("P,C", [(40000, 21), (40000, 77), (8, 150), (8, 700), (8, 1000), (1900, 3001), (8, 20001), (8, 32001), (3, 100000)])
def test_probabilities_of_equal_logits(P, C):
    """Equal logits: every exp is 1 and their sum C, both exactly, so that the gradient -p = -1/C of the labels that
    are not given has the rounding of one division alone, u relative."""
    from tt_splat_b200 import metrics
    x = torch.full((P, C), 0.75, device=DEV, requires_grad=True)
    s = metrics.label_log_probs(x, torch.zeros(P, dtype=torch.int64, device=DEV))
    (g,) = torch.autograd.grad(s.logp, x, torch.ones(P, device=DEV))
    assert (g[:, 1:].double() * -C - 1).abs().max() <= 1.01 * U


@pytest.mark.parametrize("P,C,dt", [(1300, 20001, torch.float32), (1600, 20003, torch.bfloat16), (1600, 20008, torch.float16),
                                    (2110, 33333, torch.float32), (700, 60001, torch.bfloat16)])
@pytest.mark.parametrize("aligned", [True, False])
def test_gradient_in_several_steps(P, C, dt, aligned):
    """Rows so many and so long that a block of the gradient takes several steps of 1024 16-byte vectors, the last
    block fewer; logits that line up with their gradient and columns of a wider tensor that do not.  Every element
    is compared, masked rows among them; rows without a gradient are exactly zero and change no other."""
    from tt_splat_b200 import metrics
    x, t = _inputs(P, C, dt, seed=P, masked=0.1)
    x[5::101] = -math.inf
    x[7] = 1.0
    if not aligned:
        wide = torch.full((P, C + 9), math.nan, device=DEV, dtype=dt)
        wide[:, 1:C + 1] = x
        x = wide[:, 1:C + 1]
    _check(x, t, top=2)
    torch.cuda.empty_cache()
    g = [torch.randn(P, device=DEV), torch.randn(P, device=DEV)]
    leaf = x.detach().requires_grad_(True)
    s = metrics.label_log_probs(leaf, t)
    (full,) = torch.autograd.grad([s.logp, s.entropy], leaf, g, retain_graph=True)
    for q in g:
        q[::7] = 0.0
    (some,) = torch.autograd.grad([s.logp, s.entropy], leaf, g)
    kept = torch.arange(P, device=DEV) % 7 != 0
    assert (some[~kept] == 0).all() and torch.equal(some[kept], full[kept])


def test_gradient_past_32_bits():
    """The last rows of a gradient of more than 2^31 elements, element by element: equal logits but one, so that
    p_j = 1 / S with S = C - 1 + e^8, off by 6u for the sum and its parts, and the rounding of the result."""
    from tt_splat_b200 import metrics
    C = 65536
    P = 2 ** 31 // C + 2
    x = torch.zeros(P, C, dtype=torch.float16, device=DEV)
    x[-3:, 9] = 8.0
    t = torch.full((P,), 5, dtype=torch.int64, device=DEV)
    x.requires_grad_(True)
    s = metrics.label_log_probs(x, t)
    (g,) = torch.autograd.grad(s.logp, x, torch.full((P,), 4096.0, device=DEV))
    S = C - 1 + math.exp(8.0)
    ref = torch.full((C,), -4096.0 / S, dtype=torch.float64, device=DEV)
    ref[5] += 4096.0
    ref[9] *= math.exp(8.0)
    # beside the rounding: the sum's 2 (8 + 4) u for its one large part, C / 32 + 16 additions, and 6u
    tol = ref.abs() * (torch.finfo(torch.float16).eps / 2 + (24 + C / 32 + 16 + 6) * U) + 2.0 ** -25
    assert ((g[-3:].double() - ref).abs() <= tol).all()
    assert ((g[-4].double() + 4096.0 / C)[torch.arange(C, device=DEV) != 5].abs() <= 4096.0 / C * 2.0 ** -11).all()
