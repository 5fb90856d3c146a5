"""Low-rank adapters of many requests (szh_adapters_*, szh_net_*_adapted_dev) against their plain form in float64, every
value within the bound that an f32 evaluation can be held to (tests/tracked.py)."""
import numpy as np
import pytest

import streamz_amd as sz
import tracked as tr
from helpers import _DevView, dropout_keep

pytestmark = pytest.mark.gpu


def make(rng, dims, slots, rank, n, zero_rows=True):
    i, h1, h2, o = dims
    params = [rng.uniform(-1, 1, s) * (np.sqrt(3.0 / s[0]) if len(s) == 2 else 0.1) for s in ((i, h1), (h1,), (h1, h2), (h2,), (h2, o), (o,))]
    params = [p.astype(np.float32) for p in params]
    f = [(h1, rank), (rank, h2), (h2, rank), (rank, o)]
    bank = np.concatenate([(rng.uniform(-1, 1, (slots, a * b)) / np.sqrt(a)).astype(np.float32) for a, b in f], axis=1)
    x = rng.standard_normal((n, i)).astype(np.float32)
    if zero_rows and n > 4:
        x[rng.integers(0, n, max(1, n // 20))] = 0.0
    return params, bank, x


def pick_slots(rng, n, slots, order):
    if order == "runs":
        s = np.sort(rng.integers(-1, slots, n))
        cut = rng.integers(0, n) if n > 1 else 0
        s = np.concatenate([s[cut:], s[:cut]])
    elif order == "one":
        s = np.full(n, slots - 1)
    elif order == "none":
        s = np.full(n, -1)
    else:
        s = rng.integers(-2, slots + 2, n)   # values outside the bank among them
    return s.astype(np.int32)


def known(slots, s):
    return np.where((s >= 0) & (s < slots), s, -1)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host_controls(rng, sets, out, n, allow=True, bias=True):
    c = {"sets": sets, "set_of_row": rng.integers(-1, sets + 1, n).astype(np.int32)}
    if bias:
        c["bias"] = rng.standard_normal((sets, out)).astype(np.float32)
    if allow:
        c["allow"] = rng.integers(0, 1 << 32, (sets, (out + 31) // 32), dtype=np.uint32)
        c["allow"][sets // 2] = 0   # nobody is a candidate
    return c


def dev_controls(c):
    d = {k: v if k == "sets" else dev(v.view(np.int32) if v.dtype == np.uint32 else v) for k, v in c.items()}
    return sz.LogitControls(**{k: v if k == "sets" else v.data_ptr() for k, v in d.items()}), d


def forward(net, bank, x, s, controls=None, stream=0):
    import torch
    n, out = len(x), net.output_size()
    dx, ds = dev(x), dev(s)
    logits = torch.full((n + 1, out), 7.0, device="cuda")
    probs = torch.full((n + 1, out), 7.0, device="cuda")
    net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=probs.data_ptr(), logits_ptr=logits.data_ptr(), controls=controls,
                            stream=stream)
    torch.cuda.synchronize()
    assert (logits[n] == 7).all() and (probs[n] == 7).all()   # what lies behind the last row stays
    return logits[:n].cpu().numpy(), probs[:n].cpu().numpy()


def grads(net, bank, x, labels, s, controls=None, dropout=0.0, seed=0, zero=True):
    import torch
    dx, ds, dl = dev(x), dev(s), dev(labels)
    if zero:
        bank.zero_grad_dev()
    bank.accumulate_dev(net, dx.data_ptr(), dl.data_ptr(), ds.data_ptr(), len(x), controls=controls, dropout=dropout, seed=seed)
    torch.cuda.synchronize()
    g = torch.as_tensor(_DevView(bank.grad_ptr(), bank.grad_len()), device="cuda").cpu().numpy()
    P = bank.param_count()
    return g[:bank.slots * P].reshape(bank.slots, P), g[bank.slots * P:].reshape(bank.slots, 2)


SHAPES = [
    # dims, slots, rank, rows, order
    ((60, 512, 256, 16), 4, 8, 1, "one"),
    ((60, 512, 256, 16), 4, 8, 1, "none"),
    ((60, 512, 256, 16), 64, 16, 64, "mixed"),
    ((60, 512, 256, 16), 5, 16, 700, "runs"),
    ((60, 512, 256, 16), 9, 64, 333, "mixed"),
    ((60, 512, 256, 64), 3, 1, 97, "mixed"),
    ((60, 37, 29, 3), 3, 5, 130, "mixed"),
    ((60, 33, 70, 101), 2, 17, 65, "runs"),
    ((7, 16, 8, 2), 1, 33, 31, "one"),
    ((70, 40, 24, 5), 6, 3, 515, "mixed"),
    ((60, 512, 256, 1), 2, 4, 20, "mixed"),
    ((60, 256, 512, 300), 3, 40, 260, "runs"),
]


@pytest.mark.parametrize("dims,slots,rank,n,order", SHAPES)
@pytest.mark.parametrize("controlled", [False, True])
def test_forward(dims, slots, rank, n, order, controlled):
    rng = np.random.default_rng(sum(dims) * 1000 + slots * 100 + rank + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, order)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    c = host_controls(rng, 4, dims[3], n) if controlled else None
    handle, keep = dev_controls(c) if controlled else (None, None)
    logits, probs = forward(net, bank, x, s, handle)
    want = tr.layers(params, flat, known(slots, s), 0.7, x, rank, dims)[4]
    tr.check(logits, want, "logits")
    tr.check(probs, tr.control(want, c, dims[3])[1], "probabilities")


@pytest.mark.parametrize("dims,slots,rank,n,order", SHAPES)
@pytest.mark.parametrize("controlled", [False, True])
def test_gradients(dims, slots, rank, n, order, controlled):
    rng = np.random.default_rng(sum(dims) * 1000 + slots * 100 + rank + n + 1)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, order)
    labels = rng.integers(-1, dims[3] + 1, n).astype(np.int32)   # unlabelled rows and labels that do not exist among them
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    c = host_controls(rng, 4, dims[3], n) if controlled else None
    handle, keep = dev_controls(c) if controlled else (None, None)
    g, stats = grads(net, bank, x, labels, s, handle)
    want, want_stats = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims, c)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")
    again, stats2 = grads(net, bank, x, labels, s, handle)
    assert np.array_equal(g, again) and np.array_equal(stats, stats2)


@pytest.mark.parametrize("mode", ["f32", "bf16x3"])
def test_the_large_products_and_both_arithmetic_modes(mode):
    """Enough rows for the 256-wide kernels (and for the split bf16 ones, which drop products below 2^-24 of a term: one more
    rounding per product)."""
    dims, slots, rank, n = (60, 1024, 512, 40), 7, 24, 66000
    rng = np.random.default_rng(5)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    s[:4096] = 3
    net = sz.SimpleNeuralNet(*dims, init=params)
    net.set_gemm(mode)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    logits, probs = forward(net, bank, x, s)
    part = np.concatenate([np.arange(0, 300), rng.integers(0, n, 300), np.arange(n - 300, n)])
    want = tr.layers(params, flat, known(slots, s[part]), 0.7, x[part], rank, dims)[4]
    want.e = want.e * (2 if mode == "bf16x3" else 1)
    tr.check(logits[part], want, "logits")
    # every row: the gradient over all of them is linear in row sums that a rounding cannot hide
    assert np.isfinite(logits).all() and np.abs(probs.sum(axis=1) - 1).max() < 60 * tr.U


def test_more_rows_than_one_pass():
    """Pieces of 131072 rows: rows on both sides of the border, sums over both pieces."""
    dims, slots, rank, n = (60, 64, 32, 8), 3, 4, 131072 + 77
    rng = np.random.default_rng(6)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    labels = rng.integers(0, 8, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    c = host_controls(rng, 5, 8, n)
    handle, keep = dev_controls(c)
    logits, probs = forward(net, bank, x, s, handle)
    want = tr.layers(params, flat, known(slots, s), 1.0, x, rank, dims)[4]
    tr.check(logits, want, "logits")
    tr.check(probs, tr.control(want, c, 8)[1], "probabilities")
    g, stats = grads(net, bank, x, labels, s, handle)
    want, want_stats = tr.train(params, flat, known(slots, s), 1.0, x, labels, rank, dims, c)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")


def test_a_row_does_not_depend_on_the_others():
    """The same rows alone, among others and in another order give the same bits; an adapter full of NaN and inf reaches its own rows only."""
    dims, slots, rank, n = (60, 512, 256, 16), 6, 16, 2100
    rng = np.random.default_rng(7)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    clean, _ = forward(net, bank, x, s)
    perm = rng.permutation(n)
    assert np.array_equal(forward(net, bank, x[perm], s[perm])[0], clean[perm])
    poison = [p.copy() for p in bank.get_params(2)]
    for p in poison:
        p.flat[::3] = np.nan
        p.flat[1::3] = np.inf
    bank.set_params(2, poison)
    dirty, probs = forward(net, bank, x, s)
    mine = s == 2
    assert np.array_equal(dirty[~mine], clean[~mine])
    assert np.isnan(probs[mine]).all()
    x[5] = np.nan
    assert np.array_equal(forward(net, bank, x, s)[0][~mine & (np.arange(n) != 5)], clean[~mine & (np.arange(n) != 5)])
    labels = rng.integers(0, 16, n).astype(np.int32)
    g, stats = grads(net, bank, x, labels, s)
    fine = [k for k in range(slots) if k != 2 and k != s[5]]
    assert np.isfinite(g[fine]).all() and np.isfinite(stats[fine]).all()


def test_without_adapters_it_is_the_net_itself():
    """b = 0 (a new bank) and rows without a slot: the probabilities of szh_net_forward_dev, to the rounding of another product order."""
    import torch
    dims, n = (60, 512, 256, 16), 700
    rng = np.random.default_rng(8)
    params, _, x = make(rng, dims, 1, 1, n)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, 3, 8, seed=4)
    s = pick_slots(rng, n, 3, "mixed")
    logits, probs = forward(net, bank, x, s)
    want = tr.control(tr.layers(params, np.zeros((1, 1)), np.full(n, -1), 1.0, x, 1, dims)[4], None, 16)[1]
    tr.check(probs, want)
    dx = dev(x)
    out = torch.empty(n, 16, device="cuda")
    net.forward_dev(dx.data_ptr(), n, out.data_ptr())
    torch.cuda.synchronize()
    tr.check(out.cpu().numpy(), want)


def test_dropout_is_that_of_the_net_and_keyed_by_row():
    dims, slots, rank, n = (60, 48, 32, 6), 3, 4, 200
    rng = np.random.default_rng(9)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 6, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    g, stats = grads(net, bank, x, labels, s, dropout=0.3, seed=77)
    xd = np.where(dropout_keep(77, n, 0.3), x, 0).astype(np.float32)
    want, want_stats = tr.train(params, flat, known(slots, s), 1.0, xd, labels, rank, dims)
    tr.check(stats, want_stats)
    tr.check(g, want)


def test_gradients_add_up_over_calls_and_empty_calls_do_nothing():
    dims, slots, rank, n = (60, 48, 32, 6), 3, 4, 150
    rng = np.random.default_rng(10)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 6, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    grads(net, bank, x[:60], labels[:60], s[:60])
    bank.accumulate_dev(net, 0, 0, 0, 0)
    g, stats = grads(net, bank, x[60:], labels[60:], s[60:], zero=False)
    want, want_stats = tr.train(params, flat, known(slots, s), 1.0, x, labels, rank, dims)
    tr.check(stats, tr.T(want_stats.v, want_stats.e + tr.U * want_stats.v), "stats")
    tr.check(g, tr.T(want.v, want.e + tr.U * (np.abs(want.v) + want.e)))
    net.forward_adapted_dev(bank, 0, 0, 0)


@pytest.mark.parametrize("dims,out_sets", [((60, 64, 32, 8), 3), ((60, 40, 24, 70), 2)])
def test_votes_of_many_requests(dims, out_sets):
    import torch
    slots, rank, n, groups, thr = 4, 3, 1500, 6, 0.2
    rng = np.random.default_rng(11)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, group = pick_slots(rng, n, slots, "mixed"), rng.integers(-1, groups + 1, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    c = host_controls(rng, out_sets, dims[3], n)
    handle, keep = dev_controls(c)
    _, probs = forward(net, bank, x, s, handle)
    dx, ds, dg = dev(x), dev(s), dev(group)
    counts = torch.ones(groups, dims[3], dtype=torch.int64, device="cuda")
    net.vote_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, thr, counts.data_ptr(), groups=groups, group_of_row_ptr=dg.data_ptr(), controls=handle)
    torch.cuda.synchronize()
    want = np.ones((groups, dims[3]), np.int64)
    for i in range(n):
        if 0 <= group[i] < groups and probs[i].max() > 0 and probs[i].max() >= np.float32(thr):
            want[group[i], dims[3] - 1 - int(np.argmax(probs[i][::-1]))] += 1
    assert np.array_equal(counts.cpu().numpy(), want)


def test_a_training_run_of_all_operators_together():
    """forward, loss, gradients, a norm for each adapter, clipping and update, three steps, against the plain forms step by step from the
    parameters that the run has."""
    import torch
    dims, slots, rank, n, lr, top = (60, 96, 64, 12), 5, 6, 400, 0.5, 0.05
    rng = np.random.default_rng(12)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 12, n).astype(np.int32)
    s[s == 4] = 1   # nobody uses slot 4
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.5, init=flat)
    c = host_controls(rng, 3, 12, n)
    handle, keep = dev_controls(c)
    norms = torch.zeros(slots, device="cuda")
    for _ in range(3):
        before = np.stack([np.concatenate([p.ravel() for p in bank.get_params(k)]) for k in range(slots)])
        raw, stats = grads(net, bank, x, labels, s, handle)
        want, _ = tr.train(params, before, known(slots, s), 0.5, x, labels, rank, dims, c)
        tr.check(raw, want)
        bank.clip_grad_dev(top, norms.data_ptr())
        bank.apply_grad_dev(lr)
        torch.cuda.synchronize()
        after = np.stack([np.concatenate([p.ravel() for p in bank.get_params(k)]) for k in range(slots)])
        live = stats[:, 1].astype(np.float64)
        norm = np.where(live > 0, np.sqrt((raw.astype(np.float64) ** 2).sum(axis=1)) / np.maximum(live, 1), 0)
        np.testing.assert_allclose(norms.cpu().numpy(), norm, rtol=2 * tr.U)
        f = np.where(norm > top, top / np.maximum(norm, 1e-30), 1.0)
        step = np.where(live > 0, lr / np.maximum(live, 1), 0)[:, None] * (raw * f[:, None])
        # factor, its product, lr / live, its product and the difference
        assert (np.abs(after - (before - step)) <= U5 * np.abs(step) + tr.U * np.abs(after)).all()
        assert np.array_equal(after[4], before[4])
    loss = [stats[:, 0].sum()]
    assert np.isfinite(loss).all()
    # the net itself has not moved
    assert all(np.array_equal(a, b) for a, b in zip(net.get_params(), params))


U5 = 5 * tr.U


def test_captured_and_replayed():
    """zero, accumulate, clip and forward as one graph, replayed with other inputs and with eager work of the same bank between the replays."""
    import torch
    dims, slots, rank, n = (60, 512, 256, 16), 5, 16, 900
    rng = np.random.default_rng(13)
    params, flat, x = make(rng, dims, slots, rank, n)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    bank.reserve(n, training=True)
    labels = rng.integers(0, 16, n).astype(np.int32)
    dx, ds, dl = dev(x), dev(pick_slots(rng, n, slots, "mixed")), dev(labels)
    probs, norms = torch.zeros(n, 16, device="cuda"), torch.zeros(slots, device="cuda")
    grad = torch.as_tensor(_DevView(bank.grad_ptr(), bank.grad_len()), device="cuda")

    def work(stream):
        bank.zero_grad_dev(stream)
        bank.accumulate_dev(net, dx.data_ptr(), dl.data_ptr(), ds.data_ptr(), n, stream=stream)
        bank.clip_grad_dev(0.01, norms.data_ptr(), stream)
        net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=probs.data_ptr(), stream=stream)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        work(torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        x = rng.standard_normal(x.shape).astype(np.float32)
        dx.copy_(torch.from_numpy(x))
        ds.copy_(torch.from_numpy(pick_slots(rng, n, slots, "mixed")))
        torch.cuda.synchronize()
        work(0)
        torch.cuda.synchronize()
        want = [t.clone() for t in (probs, norms, grad)]
        if k == 2:   # a larger eager call: the workspace that the graph holds must outlive it
            big = rng.standard_normal((3 * n, 60)).astype(np.float32)
            forward(net, bank, big, pick_slots(rng, 3 * n, slots, "mixed"))
        for t in (probs, norms, grad):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((probs, norms, grad), want):
            assert torch.equal(a, b)


def test_a_capture_that_would_allocate_is_refused():
    import torch
    dims, n = (60, 64, 32, 8), 300
    rng = np.random.default_rng(14)
    params, flat, x = make(rng, dims, 2, 4, n)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, 2, 4, init=flat)
    dx, ds = dev(x), dev(pick_slots(rng, n, 2, "mixed"))
    probs = torch.zeros(n, 8, device="cuda")
    side = torch.cuda.Stream()
    said = []
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        st = torch.cuda.current_stream().cuda_stream
        for call in (lambda: net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=probs.data_ptr(), stream=st),
                     lambda: bank.clip_grad_dev(1.0, 0, st), lambda: net.clip_grad_dev(1.0, 0, st)):
            with pytest.raises(sz.StreamzError) as e:
                call()
            said.append(str(e.value))
        probs.zero_()
    assert "reserve" in said[0] and all("captured" in t for t in said)


def test_another_stream():
    import torch
    dims, slots, rank, n = (60, 512, 256, 16), 5, 16, 3000
    rng = np.random.default_rng(15)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    want = forward(net, bank, x, s)
    side = torch.cuda.Stream()
    got = forward(net, bank, x, s, stream=side.cuda_stream)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_refusals():
    rng = np.random.default_rng(16)
    net = sz.SimpleNeuralNet(60, 32, 16, 4, seed=1)
    for kw, text in ((dict(slots=0, rank=4), "slots"), (dict(slots=8193, rank=1), "slots"), (dict(slots=1, rank=0), "rank"), (dict(slots=1, rank=65), "rank"),
                     (dict(slots=1, rank=1, scale=float("nan")), "scale")):
        with pytest.raises(sz.StreamzError) as e:
            sz.Adapters(net, **kw)
        assert e.value.code == -1 and text in str(e.value)
    bank = sz.Adapters(net, 2, 3)
    with pytest.raises(ValueError):
        sz.Adapters(net, 2, 3, init=np.zeros(5, np.float32))
    for call, text in ((lambda: bank.get_params(2), "slot 2 of 2"), (lambda: bank.set_params(7, bank.get_params(0)), "slot 7 of 2"),
                       (lambda: bank.clip_grad_dev(-1.0), "max_norm"), (lambda: bank.clip_grad_dev(float("nan")), "max_norm"),
                       (lambda: net.clip_grad_dev(-0.5), "max_norm"),
                       (lambda: net.forward_adapted_dev(bank, 0, 0, 4, probs_ptr=4096), "null"),
                       (lambda: net.forward_adapted_dev(bank, 4096, 4096, 4), "no result"),
                       (lambda: net.vote_adapted_dev(bank, 4096, 4096, 4, 0.5, 4096, groups=0), "group"),
                       (lambda: bank.accumulate_dev(net, 4096, 0, 4096, 4), "null"),
                       (lambda: bank.accumulate_dev(net, 4096, 4096, 4096, 4, controls=sz.LogitControls(counts=4096)), "penalties")):
        with pytest.raises(sz.StreamzError) as e:
            call()
        assert e.value.code == -1 and text in str(e.value)
    net.add_output_class(np.zeros(16, np.float32))
    d = dev(np.zeros((1, 60), np.float32))
    for call in (lambda: net.forward_adapted_dev(bank, d.data_ptr(), d.data_ptr(), 1, probs_ptr=d.data_ptr()),
                 lambda: bank.accumulate_dev(net, d.data_ptr(), d.data_ptr(), d.data_ptr(), 1)):
        with pytest.raises(sz.StreamzError) as e:
            call()
        assert "60-32-16-4" in str(e.value) and "60-32-16-5" in str(e.value)


def test_parameters_go_in_and_out():
    net = sz.SimpleNeuralNet(60, 33, 17, 5, seed=1)
    bank = sz.Adapters(net, 3, 7, seed=9)
    a2, b2, a3, b3 = bank.get_params(1)
    assert a2.shape == (33, 7) and b2.shape == (7, 17) and a3.shape == (17, 7) and b3.shape == (7, 5)
    assert not b2.any() and not b3.any() and 0 < np.abs(a2).max() <= 0.5 / np.sqrt(33) + 1e-7
    assert not np.array_equal(a2, bank.get_params(2)[0])
    new = [np.arange(p.size, dtype=np.float32).reshape(p.shape) + i for i, p in enumerate((a2, b2, a3, b3))]
    bank.set_params(1, new)
    assert all(np.array_equal(p, q) for p, q in zip(bank.get_params(1), new))
    assert np.array_equal(sz.Adapters(net, 3, 7, seed=9).get_params(2)[0], bank.get_params(2)[0])
