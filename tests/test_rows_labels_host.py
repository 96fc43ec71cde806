"""Refusals of the row lookup and the label scores, before anything reaches a GPU: wrong types, shapes
and ranges in Python, and the C entry points' own checks (null pointers are never touched)."""
import pytest
import torch


def test_gather_rows_refusals(pkg):
    from tt_splat_b200 import binned
    table, idx = torch.zeros(4, 3), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        binned.gather_rows(table, idx)
    with pytest.raises(ValueError, match="dimension"):
        binned.gather_rows(torch.zeros(()), idx)
    with pytest.raises(TypeError, match="table"):
        binned.gather_rows(table.double(), idx)
    with pytest.raises(TypeError, match="idx"):
        binned.gather_rows(table, idx.to(torch.int16))
    with pytest.raises(TypeError, match="idx"):
        binned.gather_rows(table, idx.float())
    with pytest.raises(TypeError, match="valid"):
        binned.gather_rows(table, idx, valid=torch.ones(5))
    with pytest.raises(ValueError, match="valid"):
        binned.gather_rows(table, idx, valid=torch.ones(4, dtype=torch.bool))
    with pytest.raises(TypeError, match="weight"):
        binned.gather_rows(table, idx, weight=torch.ones(5, dtype=torch.float64))
    with pytest.raises(TypeError, match="scale"):
        binned.gather_rows(table, idx, scale=torch.ones(()))
    with pytest.raises(ValueError, match="weight"):
        binned.gather_rows(table, idx, weight=torch.ones(5, 1))


def test_label_log_probs_refusals(pkg):
    from tt_splat_b200 import metrics
    x, t = torch.zeros(5, 7), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        metrics.label_log_probs(x, t)
    with pytest.raises(ValueError, match="at least one label"):
        metrics.label_log_probs(torch.zeros(5, 0), t)
    with pytest.raises(TypeError, match="logits"):
        metrics.label_log_probs(x.double(), t)
    with pytest.raises(TypeError, match="labels"):
        metrics.label_log_probs(x, t.float())
    with pytest.raises(ValueError, match="labels"):
        metrics.label_log_probs(x, t[:4])
    for top in (-1, 17):
        with pytest.raises(ValueError, match="top"):
            metrics.label_log_probs(x, t, top=top)


def test_c_entry_points_refuse(pkg):
    from tt_splat_b200 import _lib
    lib = _lib.lib()
    err = lambda: lib.tts_last_error().decode()  # noqa: E731
    gather = lambda R, C, type, N: lib.tts_gather_rows(None, R, C, C, type, None, 0, None, None, 1.0, N, None, None)  # noqa: E731
    assert gather(4, 3, 3, 5) == 1 and "type" in err()
    assert gather(4, 3, -1, 5) == 1 and "type" in err()
    assert gather(4, 3, 0, 2 ** 31) == 1 and "lookups" in err()
    assert gather(2 ** 31 - 1, 3, 0, 5) == 1 and "table rows" in err()
    assert gather(4, 2 ** 31, 0, 5) == 1 and "width" in err()
    assert gather(4, 3, 0, 5) == 1 and "null" in err()
    assert gather(4, 3, 0, 0) == 0 and gather(4, 0, 0, 5) == 0       # nothing to write
    assert lib.tts_gather_rows_bwd_workspace_bytes(1000, 100, 8) > 0
    fake = 16                                                       # never dereferenced on the host
    bwd = lambda **k: lib.tts_gather_rows_bwd(k.get("table"), 4, 3, 3, 0, k.get("idx"), 0, None, None, 1.0, 5,  # noqa: E731
                                              k.get("gout"), 3, k.get("gtable"), k.get("gweight"), None, 0, None)
    assert bwd(gtable=fake) == 1 and "null" in err()
    assert bwd(idx=fake, gout=fake, gweight=fake) == 1 and "needs the table" in err()
    assert bwd(idx=fake, gout=fake, gtable=fake) == 3 and "workspace" in err()
    assert bwd(idx=fake, gout=fake) == 0                            # no gradient wanted
    score = lambda P, C, type, top: lib.tts_label_log_probs(None, P, C, C, type, None, 0, top, None, None, None, None,  # noqa: E731
                                                            None, None)
    assert score(5, 7, 9, 0) == 1 and "type" in err()
    assert score(5, 0, 0, 0) == 1 and "labels" in err()
    assert score(2 ** 31, 7, 0, 0) == 1 and "rows" in err()
    assert score(5, 7, 0, 17) == 1 and "top" in err()
    assert score(5, 7, 0, 0) == 1 and "null" in err()
    assert score(0, 7, 0, 0) == 0
    assert lib.tts_label_log_probs_bwd(None, 5, 7, 7, 0, None, 0, 0, None, None, None, None, None, None, None, None) == 1
    assert "null" in err()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(pkg, grad):
    """A dual tensor raises whether or not a graph is recorded: a result without a tangent would read as a
    derivative of zero."""
    import torch.autograd.forward_ad as fw
    from tt_splat_b200 import binned, metrics
    table, idx, labels = torch.zeros(4, 3), torch.zeros(5, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)
    weight = torch.ones(5)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda t: fw.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))  # noqa: E731
        with pytest.raises(NotImplementedError, match="table has a forward-mode tangent"):
            binned.gather_rows(dual(table), idx)
        with pytest.raises(NotImplementedError, match="weight has a forward-mode tangent"):
            binned.gather_rows(table, idx, weight=dual(weight))
        with pytest.raises(NotImplementedError, match="logits has a forward-mode tangent"):
            metrics.label_log_probs(dual(table), labels)
        with pytest.raises(RuntimeError, match="CUDA"):
            binned.gather_rows(table, idx, weight=weight)


def test_a_lost_tile_is_named(pkg):
    """The status bit of a bulk copy that never arrived names the label scores beside the render's tiles."""
    from tt_splat_b200 import train
    assert "label scores" in train.status_message(1) and "per-tile forward" in train.status_message(1)


def test_c_entry_points_refuse_misaligned_pointers(pkg):
    """Addresses between two elements, and stats between two pairs, are refused before a launch (the addresses are
    made up: nothing reads them)."""
    from tt_splat_b200 import _lib
    lib = _lib.lib()
    refused = lambda rc: rc == 1 and "aligned" in lib.tts_last_error().decode()  # noqa: E731
    ok = 4096
    for type, e in ((0, 4), (1, 2), (2, 2)):
        def gather(table=ok, idx=ok, idx64=0, weight=None, out=ok):
            return lib.tts_gather_rows(table, 4, 3, 3, type, idx, idx64, None, weight, 1.0, 5, out, None)
        for bad in (dict(table=ok + e // 2), dict(out=ok + e // 2), dict(idx=ok + 2), dict(idx=ok + 4, idx64=1), dict(weight=ok + 2)):
            assert refused(gather(**bad)), bad

        def gather_bwd(table=ok, idx=ok, idx64=0, weight=None, gout=ok, gtable=None, gweight=None):
            return lib.tts_gather_rows_bwd(table, 4, 3, 3, type, idx, idx64, None, weight, 1.0, 5, gout, 3, gtable, gweight,
                                           ok, 1 << 30, None)
        for bad in (dict(table=ok + e // 2, gweight=ok), dict(gout=ok + e // 2, gtable=ok), dict(gtable=ok + e // 2),
                    dict(gweight=ok + 2), dict(idx=ok + 2, gtable=ok), dict(idx=ok + 4, idx64=1, gtable=ok), dict(weight=ok + 1, gtable=ok)):
            assert refused(gather_bwd(**bad)), bad

        def score(x=ok, t=ok, t64=0, logp=ok, ent=ok, tl=ok, ti=ok, stats=ok):
            return lib.tts_label_log_probs(x, 5, 7, 7, type, t, t64, 2, logp, ent, tl, ti, stats, None)
        for bad in (dict(x=ok + e // 2), dict(t=ok + 2), dict(t=ok + 4, t64=1), dict(logp=ok + 2), dict(ent=ok + 2), dict(tl=ok + 1),
                    dict(ti=ok + 4), dict(stats=ok + 4)):
            assert refused(score(**bad)), bad

        def score_bwd(x=ok, t=ok, t64=0, stats=ok, ent=ok, ti=ok, gl=ok, gh=ok, gt=ok, gx=ok):
            return lib.tts_label_log_probs_bwd(x, 5, 7, 7, type, t, t64, 2, stats, ent, ti, gl, gh, gt, gx, None)
        for bad in (dict(x=ok + e // 2), dict(gx=ok + e // 2), dict(t=ok + 2), dict(t=ok + 4, t64=1), dict(stats=ok + 4), dict(ent=ok + 2),
                    dict(ti=ok + 4), dict(gl=ok + 2), dict(gh=ok + 2), dict(gt=ok + 2)):
            assert refused(score_bwd(**bad)), bad


def test_c_entry_points_refuse_results_over_their_inputs(pkg):
    """Results in the memory of the rows that are read, whole or by one element, are refused before a launch (the
    addresses are made up: nothing reads them)."""
    from tt_splat_b200 import _lib
    lib = _lib.lib()
    refused = lambda rc: rc == 1 and "overlap" in lib.tts_last_error().decode()  # noqa: E731
    x, R, C, stride, N = 1 << 20, 4, 3, 5, 6
    for type, e in ((0, 4), (1, 2)):
        end = x + ((R - 1) * stride + C) * e                # behind the last row
        for out in (x, end - e, x - N * C * e + e):
            assert refused(lib.tts_gather_rows(x, R, C, stride, type, x - 4096, 0, None, None, 1.0, N, out, None))
        bwd = lambda table, gout, gtable: lib.tts_gather_rows_bwd(  # noqa: E731
            table, R, C, stride, type, x - 4096, 0, None, None, 1.0, N, gout, stride, gtable, None, x - 8192, 1 << 30, None)
        for gtable in (x, end - e, x - R * C * e + e):
            assert refused(bwd(x, x + 4096, gtable))
            assert refused(bwd(None, x, gtable))
        for gx in (x, end - e, x - R * C * e + e):
            assert refused(lib.tts_label_log_probs_bwd(x, R, C, stride, type, x - 4096, 0, 0, x - 8192, x - 8192, None,
                                                       x - 8192, None, None, gx, None))
