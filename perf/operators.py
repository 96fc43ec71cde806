"""Timed cases of two operators: the lookup of table rows through slot tables, with its gradient
(``binned.gather_rows``), and the log probabilities of labels with their entropy and best
alternatives, with their gradient (``metrics.label_log_probs``).

``own`` selects what ``run`` does: the operators in elementary torch operations (False), or the
framework's calls (True).  Sizes follow the framework's scenes (tiles of 16x16 pixels with 128 or
256 slots, 2k to 1M gaussians, images of 1264x832 and 800x800) or are generic vocabularies.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _rows(name, T, K, R, C, type, ids, train, index="i64", valid=False, weight=False, scale=1.0):
    return dict(name=name, op="rows", T=T, K=K, R=R, C=C, type=type, ids=ids, train=train, index=index, valid=valid,
                weight=weight, scale=scale)


def _labels(name, P, C, type, top, train, masked=False, unlabelled=0.0, index="i64", grad_top=False):
    return dict(name=name, op="labels", P=P, C=C, type=type, top=top, train=train, masked=masked, unlabelled=unlabelled,
                index=index, grad_top=grad_top)


def listed():
    return [
        # a single tile's slots looking up colours: a viewer's probe of one tile, latency alone
        _rows("rows_one_tile", 1, 128, 2000, 3, "f32", "tiles", False, valid=True),
        # per-gaussian features of one 1264x832 view gathered for a render, culled slots weighted
        _rows("rows_view_features", 4108, 128, 100000, 16, "f32", "tiles", False, valid=True, weight=True),
        # SH rows (15 x 3) of an 800x800 view in training, with a weight per slot that is learned too
        _rows("rows_sh_train", 2500, 128, 10000, 45, "f32", "tiles", True, valid=True, weight=True),
        # features of the largest scene in 16 bits: 1M gaussians, 1920x1072, 256 slots, -1 in unused slots
        _rows("rows_scene_train", 8040, 256, 1000000, 32, "bf16", "tiles", True, index="i32"),
        # tokens of a text batch: few rows with most of the uses, wide rows, one scale for all
        _rows("rows_tokens_train", 1, 8191, 32000, 1024, "bf16", "zipf", True, scale=32.0),
        # a small codebook shared by every gaussian of a scene: long sums for each row
        _rows("rows_codebook_train", 1, 100000, 512, 45, "f16", "even", True, index="i32", weight=True),
        # one row over a vocabulary: a single answer, latency alone
        _labels("labels_one", 1, 32000, "bf16", 8, False),
        # the labels of every pixel of a 1264x832 render, few classes
        _labels("labels_image", 1264 * 832, 21, "f32", 3, False, index="i32"),
        # training on an 800x800 label image, most pixels labelled
        _labels("labels_image_train", 800 * 800, 150, "bf16", 0, True, unlabelled=0.25),
        # training over a vocabulary of odd size, the alternatives' scores pulled too (distillation)
        _labels("labels_vocab_train", 4095, 32001, "f32", 4, True, grad_top=True),
        # a batch of answers over a large vocabulary
        _labels("labels_batch", 64, 131072, "f16", 16, False),
        # training with a mask of allowed labels for each row; some rows allow none
        _labels("labels_masked_train", 10007, 1000, "f32", 5, True, masked=True, unlabelled=0.1, index="i32"),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    return max(lo, min(hi, n))


def draw(rng):
    top_bytes = {op: max(work(c)["bytes"] for c in listed() if c["op"] == op) for op in ("rows", "labels")}
    top_flops = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("rows", "labels")}
    while True:
        type = rng.choice(sorted(TYPES))
        index = rng.choice(["i32", "i64"])
        if rng.random() < 0.5:
            K = rng.choice([1, 128, 256, _log_int(rng, 1, 300)])
            T = _log_int(rng, 1, 8192)
            case = _rows("", T, K, _log_int(rng, 1, 1000000), _log_int(rng, 1, 2048), type,
                         rng.choice(["tiles", "zipf", "even"]), rng.random() < 0.6, index, rng.random() < 0.5,
                         rng.random() < 0.5, rng.choice([1.0, 0.125, 5.5]))
        else:
            train = rng.random() < 0.6
            top = rng.choice([0, 1, 4, 8, 16])
            case = _labels("", _log_int(rng, 1, 1100000), _log_int(rng, 2, 131072), type, top, train,
                           rng.random() < 0.3, rng.choice([0.0, 0.1, 0.6]), index, train and top > 0 and rng.random() < 0.5)
        w = work(case)
        if case["op"] == "rows" and case["R"] * case["C"] > 1 << 28:
            continue
        if w["bytes"] <= top_bytes[case["op"]] and w["flops"] <= top_flops[case["op"]]:
            del case["name"]
            return case


def work(case):
    e = SIZES[case["type"]]
    i = 4 if case["index"] == "i32" else 8
    if case["op"] == "rows":
        N, R, C = case["T"] * case["K"], case["R"], case["C"]
        touched = min(N, R) * C * e
        nb = N * i + N * case["valid"] + 4 * N * case["weight"] + touched + N * C * e
        fl = N * C
        if case["train"]:
            nb += N * C * e + R * C * e + 4 * N * case["weight"]
            fl += 2 * N * C + 2 * N * C * case["weight"]
        return {"bytes": nb, "flops": fl}
    P, C, k = case["P"], case["C"], case["top"]
    nb = P * C * e + P * i + 8 * P + 12 * P * k
    fl = 8 * P * C
    if case["train"]:
        nb += P * C * e + 8 * P + 4 * P * k * case["grad_top"]
        fl += 6 * P * C
    return {"bytes": nb, "flops": fl}


# ---- inputs ---------------------------------------------------------------------------------


def _make_rows(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    T, K, R, C = case["T"], case["K"], case["R"], case["C"]
    dt = TYPES[case["type"]]
    it = torch.int32 if case["index"] == "i32" else torch.int64
    u = torch.rand(T, K, generator=g, device="cuda", dtype=torch.float64)
    if case["ids"] == "tiles":
        # a tile sees the gaussians around it: its own share of the ids and those of eight tiles near it
        span = min(R, max(9 * R // max(T, 9), 2 * K))
        start = torch.arange(T, device="cuda", dtype=torch.float64)[:, None] * (R / T)
        order = torch.randperm(R, generator=g, device="cuda")
        ids = order[((start + u * span).long() % R)]
    elif case["ids"] == "zipf":
        # the n-th row is used about 1/n times as often as the first
        ids = (torch.exp(u * math.log(R + 1.0)).long() - 1).clamp_(0, R - 1)
        ids = torch.randperm(R, generator=g, device="cuda")[ids]
    else:
        ids = (u * R).long().clamp_(0, R - 1)
    # a tile fills its slots from the front: most are full, some are not
    count = (torch.rand(T, 1, generator=g, device="cuda") * 1.6 * K).long() + K // 8
    used = torch.arange(K, device="cuda")[None, :] < count
    if case["ids"] != "tiles":
        used = torch.ones_like(used)
    st = dict(case=case, valid=None, weight=None)
    if case["valid"]:
        ids, st["valid"] = torch.where(used, ids, torch.zeros_like(ids)), used
    else:
        ids = torch.where(used, ids, torch.full_like(ids, -1))
    if T == 1:
        ids = ids[0]
        st["valid"] = st["valid"][0] if case["valid"] else None
    st["idx"] = ids.to(it).contiguous()
    st["table"] = torch.randn(R, C, generator=g, device="cuda").to(dt)
    if case["weight"]:
        st["weight"] = torch.rand(ids.shape, generator=g, device="cuda")
    if case["train"]:
        st["table"].requires_grad_(True)
        if case["weight"]:
            st["weight"].requires_grad_(True)
        st["gout"] = (torch.randn(ids.shape + (C,), generator=g, device="cuda") * 0.1).to(dt)
    return st


def _make_labels(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    P, C = case["P"], case["C"]
    dt = TYPES[case["type"]]
    x = torch.randn(P, C, generator=g, device="cuda")
    x.mul_(2.0)
    # a confident row has a few labels far above the rest
    best = torch.randint(0, C, (P,), generator=g, device="cuda")
    x[torch.arange(P, device="cuda"), best] += torch.rand(P, generator=g, device="cuda") * 12.0
    labels = torch.where(torch.rand(P, generator=g, device="cuda") < 0.7, best,
                         torch.randint(0, C, (P,), generator=g, device="cuda"))
    if case["masked"]:
        # each row allows its own share of the labels, and one row in 64 none
        share = torch.rand(P, 1, generator=g, device="cuda")
        share[torch.rand(P, 1, generator=g, device="cuda") < 1 / 64] = 0.0
        x.masked_fill_(torch.rand(P, C, generator=g, device="cuda") >= share, -math.inf)
        del share
    labels[torch.rand(P, generator=g, device="cuda") < case["unlabelled"]] = -1
    st = dict(case=case, logits=x.to(dt), labels=labels.to(torch.int32 if case["index"] == "i32" else torch.int64))
    if case["train"]:
        st["logits"].requires_grad_(True)
        st["g_logp"] = -torch.rand(P, generator=g, device="cuda")
        st["g_entropy"] = torch.randn(P, generator=g, device="cuda") * 0.01
        if case["grad_top"]:
            st["g_top"] = torch.randn(P, case["top"], generator=g, device="cuda") * 0.1
    return st


def prepare(case, seed):
    return _make_rows(case, seed) if case["op"] == "rows" else _make_labels(case, seed)


# ---- one pass -------------------------------------------------------------------------------


def run(state):
    if own:
        return _own_rows(state) if state["case"]["op"] == "rows" else _own_labels(state)
    with torch.no_grad():
        return _plain_rows(state) if state["case"]["op"] == "rows" else _plain_labels(state)


def _own_rows(st):
    from __graft_entry__ import load_package
    load_package()
    from tt_splat_b200 import binned
    case = st["case"]
    out = binned.gather_rows(st["table"], st["idx"], valid=st["valid"], weight=st["weight"], scale=case["scale"])
    if not case["train"]:
        return {"out": out}
    wrt = [st["table"]] + ([st["weight"]] if case["weight"] else [])
    grads = torch.autograd.grad(out, wrt, st["gout"])
    return dict(zip(("out", "gtable", "gweight"), (out.detach(), *grads)))


def _own_labels(st):
    from __graft_entry__ import load_package
    load_package()
    from tt_splat_b200 import metrics
    case = st["case"]
    s = metrics.label_log_probs(st["logits"], st["labels"], top=case["top"])
    res = {"logp": s.logp.detach(), "entropy": s.entropy.detach(), "top_logp": s.top_logp.detach(), "top_ids": s.top_ids}
    if case["train"]:
        outs, gs = [s.logp, s.entropy], [st["g_logp"], st["g_entropy"]]
        if case["grad_top"]:
            outs, gs = outs + [s.top_logp], gs + [st["g_top"]]
        (res["glogits"],) = torch.autograd.grad(outs, [st["logits"]], gs)
    return res


def _plain_rows(st):
    case, table, idx = st["case"], st["table"], st["idx"].long()
    dt, R, C = table.dtype, case["R"], case["C"]
    used = idx >= 0
    if st["valid"] is not None:
        used = used & st["valid"]
    f = used.float() * case["scale"]
    if st["weight"] is not None:
        f = f * st["weight"]
    safe = torch.where(used, idx, torch.zeros_like(idx)).reshape(-1)
    rows = table[safe].float()
    f = f.reshape(-1, 1)
    res = {"out": (rows * f).to(dt).reshape(idx.shape + (C,))}
    if case["train"]:
        go = st["gout"].reshape(-1, C).float()
        acc = torch.zeros(R, C, device=table.device)
        acc.index_add_(0, safe, go * f)
        res["gtable"] = acc.to(dt)
        if case["weight"]:
            gw = (go * rows).sum(1) * (used.reshape(-1).float() * case["scale"])
            res["gweight"] = gw.reshape(idx.shape)
    return res


def _plain_labels(st):
    case, x, labels = st["case"], st["logits"].float(), st["labels"].long()
    P, C, k = case["P"], case["C"], case["top"]
    inf = math.inf
    m = x.max(1, keepdim=True).values
    empty = m == -inf
    d = x - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    logS = torch.where(empty, torch.zeros_like(S), torch.log(S))
    p = e / torch.where(empty, torch.ones_like(S), S)
    H = logS - torch.where(p > 0, p * d, torch.zeros_like(p)).sum(1, keepdim=True)
    H = torch.where(empty, torch.zeros_like(H), H)
    lp = d - logS
    known = labels >= 0
    safe = torch.where(known, labels, torch.zeros_like(labels))[:, None]
    logp = torch.where(known, lp.gather(1, safe)[:, 0], torch.zeros_like(H[:, 0]))
    ids = torch.full((P, k), -1, dtype=torch.int64, device=x.device)
    tlp = torch.full((P, k), -inf, device=x.device)
    rest = lp.clone() if k else None
    raw = x.clone() if k else None
    for j in range(min(k, C)):
        best, at = raw.max(1)
        ok = best > -inf
        ids[:, j] = torch.where(ok, at, torch.full_like(at, -1))
        tlp[:, j] = torch.where(ok, rest.gather(1, at[:, None])[:, 0], tlp[:, j])
        raw.scatter_(1, at[:, None], -inf)
    res = {"logp": logp, "entropy": H[:, 0], "top_logp": tlp, "top_ids": ids}
    if case["train"]:
        gl = torch.where(known, st["g_logp"], torch.zeros_like(H[:, 0]))[:, None]
        gl = torch.where(empty, torch.zeros_like(gl), gl)
        gh = st["g_entropy"][:, None]
        total = gl
        if case["grad_top"]:
            gt = torch.where(ids >= 0, st["g_top"], torch.zeros_like(tlp))
            total = total + gt.sum(1, keepdim=True)
        gx = torch.where(p > 0, p * (-total - gh * (lp + H)), torch.zeros_like(p))
        gx.scatter_add_(1, safe, gl)
        if case["grad_top"]:
            gx.scatter_add_(1, ids.clamp(min=0), gt)
        res["glogits"] = gx.to(st["logits"].dtype)
    return res


# ---- the definition in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_rows(st) if case["op"] == "rows" else _exact_labels(st)


def _exact_rows(st):
    case = st["case"]
    shape, C, R = st["idx"].shape, case["C"], case["R"]
    idx = st["idx"].reshape(-1).long()
    keep = idx >= 0 if st["valid"] is None else (idx >= 0) & st["valid"].reshape(-1)
    n = keep.nonzero()[:, 0]
    at = idx[n]
    f = torch.full((n.numel(),), float(case["scale"]), dtype=torch.float64, device=idx.device)
    if st["weight"] is not None:
        f *= st["weight"].detach().reshape(-1)[n].double()
    table = st["table"].detach().double()
    out = torch.zeros(idx.numel(), C, dtype=torch.float64, device=idx.device)
    out[n] = f[:, None] * table[at]
    res = {"out": out.reshape(shape + (C,))}
    if case["train"]:
        go = st["gout"].reshape(-1, C)[n].double()
        order = torch.argsort(at, stable=True)
        gt = torch.zeros(R, C, dtype=torch.float64, device=idx.device)
        gt.index_put_((at[order],), (f[:, None] * go)[order], accumulate=True)
        res["gtable"] = gt
        if case["weight"]:
            gw = torch.zeros(idx.numel(), dtype=torch.float64, device=idx.device)
            gw[n] = case["scale"] * torch.einsum("nc,nc->n", go, table[at])
            res["gweight"] = gw.reshape(shape)
    return res


def _exact_labels(st):
    case = st["case"]
    P, C, k = case["P"], case["C"], case["top"]
    step = max(1, min(P, 50_000_000 // C))
    parts = []
    for a in range(0, P, step):
        x = st["logits"].detach()[a:a + step].double()
        t = st["labels"][a:a + step].long()
        rows = torch.arange(x.shape[0], device=x.device)
        some = torch.isfinite(x).any(1)
        lse = torch.where(some, torch.logsumexp(x, 1), torch.zeros((), dtype=x.dtype, device=x.device))
        logq = x - lse[:, None]
        q = torch.exp(logq)
        H = -torch.special.xlogy(q, q).sum(1)
        H = torch.where(some, H, torch.zeros_like(H))
        logp = torch.where(t >= 0, logq[rows, t.clamp(min=0)], torch.zeros_like(H))
        part = {"logp": logp, "entropy": H}
        order = torch.sort(x, dim=1, descending=True, stable=True)
        kk = min(k, C)
        tid = torch.full((x.shape[0], k), -1, dtype=torch.int64, device=x.device)
        tlp = torch.full((x.shape[0], k), -math.inf, dtype=x.dtype, device=x.device)
        real = order.values[:, :kk] > -math.inf
        tid[:, :kk] = torch.where(real, order.indices[:, :kk], tid[:, :kk])
        tlp[:, :kk] = torch.where(real, order.values[:, :kk] - lse[:, None], tlp[:, :kk])
        part["top_logp"], part["top_ids"] = tlp, tid
        del order
        if case["train"]:
            # the chain rule, output by output: rows of the Jacobian are onehot - q, and
            # -q (log q + H) for the entropy
            up = torch.zeros_like(x)
            gl = st["g_logp"][a:a + step].double()
            sel = (t >= 0) & some
            up[rows[sel], t[sel]] += gl[sel]
            if case["grad_top"]:
                gk = st["g_top"][a:a + step].double()
                for j in range(k):
                    s = tid[:, j] >= 0
                    up[rows[s], tid[s, j]] += gk[s, j]
            gx = up - q * up.sum(1, keepdim=True)
            gx -= st["g_entropy"][a:a + step].double()[:, None] * (torch.special.xlogy(q, q) + q * H[:, None])
            gx[~some] = 0.0
            part["glogits"] = gx
        parts.append(part)
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
