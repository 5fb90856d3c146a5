"""Gradient norms over many tensors with their clipping (szh_clip_*, szh_net_clip_grad_dev) and the controls on logits
(szh_logits_control_dev) against float64."""
import numpy as np
import pytest

import streamz_amd as sz
import tracked as tr
from helpers import grad_view

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- clipping ------------------------------------------------------------------------------------------------

LISTS = [[1], [0], [0, 5, 0], [3, 1, 4, 1, 5, 9, 2, 6], [4096], [4097, 4095], [100_003], [7] * 300, [1_500_000, 3, 70_001, 2_000_000], [1023, 1025, 1 << 14] * 40]


@pytest.mark.parametrize("lengths", LISTS, ids=lambda v: f"{len(v)}x{max(v)}")
@pytest.mark.parametrize("how", ["one", "each", "some", "in place"])
def test_clip_many_tensors(lengths, how):
    import torch
    rng = np.random.default_rng(len(lengths) + max(lengths))
    # one buffer, tensors at odd offsets: most of them not 16-byte aligned
    total = sum(lengths) + 3 * len(lengths) + 1
    host = rng.standard_normal(total).astype(np.float32)
    buf, out = dev(host), dev(np.full(total, 7.0, np.float32))
    at, off = 1, []
    for n in lengths:
        off.append(at)
        at += n + 3
    groups = None if how in ("one", "in place") else list(range(len(lengths))) if how == "each" else [int(g) for g in rng.integers(0, 3, len(lengths))]
    gr = np.zeros(len(lengths), int) if groups is None else np.array(groups)
    ng = int(gr.max()) + 1
    live = rng.integers(1, 9, ng).astype(np.float32)
    live[0] = 4.0
    dlive, norms = dev(live), torch.full((ng + 1,), 5.0, device="cuda")
    base = buf.data_ptr()
    clip = sz.GradClip([(base + 4 * o, n) for o, n in zip(off, lengths)], groups=groups, live=dlive.data_ptr(),
                       outputs=None if how == "in place" else [out.data_ptr() + 4 * o for o in off])
    want_norm = np.array([np.sqrt(sum((host[o:o + n].astype(np.float64) ** 2).sum() for o, n, g in zip(off, lengths, gr) if g == k)) / live[k] for k in range(ng)])
    limit = float(np.float32(0.6 * np.median(want_norm)))
    clip.run(limit, norms.data_ptr())
    torch.cuda.synchronize()
    got = norms.cpu().numpy()
    assert got[ng] == 5.0
    assert (np.abs(got[:ng] - want_norm) <= 2 * tr.U * want_norm).all()
    want = np.full(total, 7.0) if how != "in place" else host.astype(np.float64)
    for o, n, g in zip(off, lengths, gr):
        want[o:o + n] = host[o:o + n] * (limit / want_norm[g] if want_norm[g] > limit else 1.0)
    res = (buf if how == "in place" else out).cpu().numpy()
    assert (np.abs(res - want) <= 2 * tr.U * np.abs(want)).all()   # the factor's rounding and the product's
    if how != "in place":
        assert np.array_equal(buf.cpu().numpy(), host)


def test_clip_values_at_the_ends_of_the_range():
    import torch
    for v, limit in ((3e38, 1.0), (1e-38, 0.5e-38), (1e-42, 1e-43)):
        g = torch.full((1000,), v, device="cuda")
        norms = torch.zeros(1, device="cuda")
        clip = sz.GradClip([(g.data_ptr(), 1000)])
        x = float(g[0].double())
        clip.run(limit, norms.data_ptr())
        torch.cuda.synchronize()
        norm = np.sqrt(1000.0) * x
        lim = float(np.float32(limit))
        assert norms.item() == np.float32(norm) or abs(norms.item() - norm) <= 2 * tr.U * norm
        want = x * (lim / norm)
        # results below the normal range are whole steps of 2^-149
        assert abs(float(g[7].double()) - want) <= 2 * tr.U * want + 2.0 ** -149


def test_clip_without_need_with_nothing_counted_and_with_values_that_are_none():
    import torch
    rng = np.random.default_rng(3)
    host = rng.standard_normal(5000).astype(np.float32)
    for live, limit, keep in ((1.0, 1e6, True), (0.0, 1e-6, True), (1.0, 0.0, False)):
        g, l, norms = dev(host), dev(np.array([live], np.float32)), torch.zeros(1, device="cuda")
        clip = sz.GradClip([(g.data_ptr(), 5000)], live=l.data_ptr())
        clip.run(limit, norms.data_ptr())
        torch.cuda.synchronize()
        assert np.array_equal(g.cpu().numpy(), host if keep else np.zeros_like(host))
        assert (norms.item() == 0.0) == (live == 0.0)
    host[17] = np.nan   # the norm is NaN: nothing is scaled, and the caller sees it
    g, norms = dev(host), torch.zeros(1, device="cuda")
    clip = sz.GradClip([(g.data_ptr(), 5000)])
    clip.run(0.1, norms.data_ptr())
    torch.cuda.synchronize()
    assert np.isnan(norms.item()) and np.array_equal(g.cpu().numpy(), host, equal_nan=True)
    host[17] = np.inf   # the norm is infinite: the factor is 0
    g = dev(host)
    clip = sz.GradClip([(g.data_ptr(), 5000)])
    clip.run(0.1, norms.data_ptr())
    torch.cuda.synchronize()
    got = g.cpu().numpy()
    assert np.isinf(norms.item()) and np.isnan(got[17]) and not np.delete(got, 17).any()


def test_clip_is_the_same_on_every_run_and_in_a_graph():
    import torch
    rng = np.random.default_rng(4)
    src = [dev(rng.standard_normal(n).astype(np.float32)) for n in (33333, 7, 120000)]
    dst = [torch.zeros_like(t) for t in src]
    norms = torch.zeros(1, device="cuda")
    clip = sz.GradClip([(t.data_ptr(), t.numel()) for t in src], outputs=[t.data_ptr() for t in dst])
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        clip.run(1.0, norms.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in src:
            t.mul_(1.5)
        clip.run(1.0, norms.data_ptr())
        torch.cuda.synchronize()
        want = [t.clone() for t in dst] + [norms.clone()]
        for t in dst + [norms]:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(dst + [norms], want))


def test_clip_between_the_sum_and_the_update_of_a_net():
    """zero_grad, accumulate, clip, apply of a net, a second class count included (its gradient vector moves)."""
    import torch
    rng = np.random.default_rng(5)
    net = sz.SimpleNeuralNet(60, 64, 32, 5, seed=3)
    x = dev(rng.standard_normal((500, 60)).astype(np.float32))
    for out in (5, 6):
        labels = dev(rng.integers(0, out, 500).astype(np.int32))
        norm = torch.zeros(1, device="cuda")
        net.zero_grad_dev()
        net.accumulate_dev(x.data_ptr(), labels.data_ptr(), 500)
        torch.cuda.synchronize()
        raw = grad_view(net).cpu().numpy().copy()
        before = net.get_flat()
        want = np.sqrt((raw[:-2].astype(np.float64) ** 2).sum()) / raw[-1]
        limit = float(np.float32(0.25 * want))
        net.clip_grad_dev(limit, norm.data_ptr())
        torch.cuda.synchronize()
        g = grad_view(net).cpu().numpy()
        assert abs(norm.item() - want) <= 2 * tr.U * want
        assert np.array_equal(g[-2:], raw[-2:])
        assert (np.abs(g[:-2] - raw[:-2] * (limit / want)) <= 2 * tr.U * np.abs(g[:-2])).all()
        net.apply_grad_dev(0.5)
        step = 0.5 / raw[-1] * g[:-2].astype(np.float64)
        assert (np.abs(net.get_flat() - (before - step)) <= 3 * tr.U * np.abs(step) + tr.U * np.abs(before - step) + 1e-30).all()
        net.add_output_class(np.zeros(32, np.float32))


# ---- controls ------------------------------------------------------------------------------------------------

def host_controls(rng, sets, classes, rows, parts):
    c = {"sets": sets, "set_of_row": rng.integers(-1, sets + 1, rows).astype(np.int32)}
    if "bias" in parts:
        c["bias"] = rng.standard_normal((sets, classes)).astype(np.float32)
    if "allow" in parts:
        c["allow"] = rng.integers(0, 1 << 32, (sets, (classes + 31) // 32), dtype=np.uint32)
        c["allow"][-1] = 0
    if "counts" in parts:
        c["counts"] = np.maximum(rng.integers(-20, 9, (sets, classes)), 0).astype(np.uint32)
        c["repetition"] = rng.uniform(0.5, 2.0, sets).astype(np.float32)
        c["presence"] = rng.uniform(-1, 1, sets).astype(np.float32)
        c["frequency"] = rng.uniform(-0.2, 0.2, sets).astype(np.float32)
    return c


def run_controls(logits, c, ld_in, ld_out, probs, in_place=False):
    import torch
    rows, classes = logits.shape
    src = torch.full((rows, ld_in), 3.0, device="cuda")
    src[:, :classes] = dev(logits)
    out = src if in_place else torch.full((rows, ld_out), 7.0, device="cuda")
    keep = {} if c is None else {k: v if k == "sets" else dev(v.view(np.int32) if v.dtype == np.uint32 else v) for k, v in c.items()}
    handle = None if c is None else sz.LogitControls(**{k: v if k == "sets" else v.data_ptr() for k, v in keep.items()})
    sz.control_logits_dev(src.data_ptr(), rows, classes, handle, out.data_ptr(), probs=probs, ld_logits=ld_in, ld_out=ld_in if in_place else ld_out)
    torch.cuda.synchronize()
    if not in_place:
        assert (out[:, classes:] == 7.0).all() and np.array_equal(src[:, :classes].cpu().numpy(), logits, equal_nan=True)
    else:
        assert (out[:, classes:] == 3.0).all()
    return out[:, :classes].cpu().numpy()


PARTS = [(), ("bias",), ("allow",), ("counts",), ("bias", "allow", "counts")]


@pytest.mark.parametrize("classes", [1, 2, 3, 15, 16, 31, 33, 64, 65, 100, 128, 255, 256, 257, 1000, 1025, 4097, 20000])
@pytest.mark.parametrize("parts", PARTS, ids=lambda p: "+".join(p) or "none")
def test_controls(classes, parts):
    rng = np.random.default_rng(classes * 7 + len(parts))
    rows = 301 if classes < 1000 else 37
    logits = (4 * rng.standard_normal((rows, classes))).astype(np.float32)
    c = host_controls(rng, 5, classes, rows, parts) if parts else None
    z, p = tr.control(tr.T(logits), c, classes)
    tr.check(run_controls(logits, c, classes, classes, True), p, "probabilities")
    tr.check(run_controls(logits, c, classes + 3, classes + 5, False), z, "logits")
    tr.check(run_controls(logits, c, classes + 1, 0, True, in_place=True), p, "in place")


@pytest.mark.parametrize("classes", [70001, 140000])
def test_controls_of_very_many_classes(classes):
    rng = np.random.default_rng(classes)
    logits = (4 * rng.standard_normal((5, classes))).astype(np.float32)
    c = host_controls(rng, 3, classes, 5, PARTS[-1])
    z, p = tr.control(tr.T(logits), c, classes)
    tr.check(run_controls(logits, c, classes, classes, True), p)
    tr.check(run_controls(logits, c, classes, classes, False), z)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 100_001])
def test_controls_rows_and_shared_set(rows):
    rng = np.random.default_rng(rows)
    logits = (4 * rng.standard_normal((rows, 16))).astype(np.float32)
    c = host_controls(rng, 1, 16, rows, PARTS[-1])
    c["allow"][0] = 0x00f3
    del c["set_of_row"]
    tr.check(run_controls(logits, c, 16, 16, True), tr.control(tr.T(logits), c, 16)[1])


@pytest.mark.parametrize("classes", [5, 16, 64, 70, 700, 6000])
def test_controls_of_values_that_are_none(classes):
    rng = np.random.default_rng(classes + 1)
    logits = rng.standard_normal((8, classes)).astype(np.float32)
    allow = np.full((3, (classes + 31) // 32), 0xffffffff, np.uint32)
    allow[1, 0] = 0xfffffff8   # classes 0, 1 and 2 are out
    allow[2] = 0
    c = {"sets": 3, "allow": allow, "set_of_row": np.array([0, 1, 2, 0, 1, 1, 0, 1], np.int32)}
    logits[0, 1] = np.nan            # an allowed NaN takes its row with it
    logits[1, :3] = np.nan, np.inf, -np.inf   # outside the list: nothing happens
    logits[2, 0] = np.nan
    logits[3, 2] = -np.inf           # an allowed -inf has no probability
    logits[4, :] = -np.inf           # nothing is left
    logits[5, 3:] = np.finfo(np.float32).min   # the type's lowest value is a value like others
    logits[6, 3] = np.inf
    logits[7, 3:] = 3e38
    got = run_controls(logits, c, classes, classes, True)
    assert np.isnan(got[0]).all() and np.isnan(got[6]).all()
    assert not got[2].any() and not got[4].any()
    for i in (1, 5, 7):
        assert not got[i, :3].any() and abs(got[i].sum(dtype=np.float64) - 1) < (classes + 4) * tr.U
    assert got[3, 2] == 0 and abs(got[3].sum(dtype=np.float64) - 1) < (classes + 4) * tr.U
    z = run_controls(logits, c, classes, classes, False)
    assert np.isneginf(z[1, :3]).all() and np.isneginf(z[2]).all() and np.array_equal(z[1, 3:], logits[1, 3:])


def test_controls_captured():
    import torch
    rng = np.random.default_rng(9)
    logits = dev(rng.standard_normal((1000, 64)).astype(np.float32))
    out = torch.zeros_like(logits)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        sz.control_logits_dev(logits.data_ptr(), 1000, 64, None, out.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        logits.mul_(1.25)
        sz.control_logits_dev(logits.data_ptr(), 1000, 64, None, out.data_ptr())
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
