"""Low-rank adapters, clipping and controls where one way of computing them ends and another begins: row counts, ranks, widths and
alignments on both sides of each border, against the plain forms of tests/tracked.py; values that are none; two banks at once."""
import numpy as np
import pytest

import streamz_amd as sz
import tracked as tr
from helpers import dropout_keep
from test_gpu_adapters import dev, dev_controls, forward, grads, host_controls, known, make, pick_slots

pytestmark = pytest.mark.gpu

BORDERS = [
    # dims, slots, rank, rows, order: rows that go one by one, or in tiles
    ((60, 512, 256, 16), 6, 16, 256, "mixed"),
    ((60, 512, 256, 16), 6, 16, 257, "mixed"),
    ((60, 128, 64, 16), 6, 16, 512, "mixed"),
    ((60, 128, 64, 16), 6, 16, 513, "mixed"),
    # the first layer with its rank columns, or one after the other
    ((60, 512, 64, 8), 5, 16, 601, "runs"),
    ((60, 512, 64, 8), 5, 17, 601, "runs"),
    ((60, 513, 64, 8), 5, 16, 601, "runs"),
    ((64, 100, 64, 8), 5, 3, 530, "mixed"),
    ((65, 100, 64, 8), 5, 3, 530, "mixed"),
    ((61, 65, 64, 8), 40, 9, 530, "mixed"),
    ((3, 1, 5, 2), 2, 1, 530, "mixed"),
    ((60, 64, 48, 4), 3, 8, 5000, "none"),
    # output layers of one pass, or of a product of their own
    ((60, 96, 72, 64), 4, 20, 600, "mixed"),
    ((60, 96, 72, 65), 4, 20, 600, "mixed"),
    ((60, 96, 72, 300), 4, 20, 200, "mixed"),
    ((60, 96, 300, 300), 4, 20, 40, "mixed"),
    # the output layer and back in one launch, or not; w3 streamed by every row, or not
    ((60, 70, 50, 16), 4, 16, 300, "mixed"),
    ((60, 70, 50, 17), 4, 15, 300, "mixed"),
    ((60, 70, 50, 33), 300, 16, 400, "mixed"),
    ((60, 70, 50, 64), 4, 16, 290, "runs"),
    ((60, 70, 1100, 64), 4, 9, 100, "mixed"),
    ((60, 70, 1100, 63), 4, 20, 100, "mixed"),
    # rows put in the order of their slots by one workgroup, or by four launches
    ((60, 32, 16, 4), 5, 4, 8192, "mixed"),
    ((60, 32, 16, 4), 5, 4, 8193, "mixed"),
    ((60, 32, 16, 4), 1000, 2, 1500, "mixed"),
    ((60, 32, 16, 4), 1001, 2, 1500, "mixed"),
    ((60, 32, 16, 4), 8192, 1, 700, "mixed"),
    # hidden products of whole rounds of wide tiles with a few rows behind them
    ((60, 256, 2048, 3), 7, 40, 8197, "runs"),
    ((60, 256, 2048, 3), 7, 16, 8192, "mixed"),
    ((60, 256, 2048, 3), 7, 16, 7990, "runs"),
    # ... of whole rounds of other tiles, and of both
    ((60, 1024, 2048, 4), 6, 16, 1056, "mixed"),
    ((60, 512, 2048, 3), 5, 8, 9248, "runs"),
    # few rows of many slots, chunk by chunk
    ((60, 70, 50, 20), 90, 5, 130, "mixed"),
    ((60, 70, 50, 21), 400, 19, 250, "mixed"),
    ((60, 30, 3, 2), 5, 2, 90, "mixed"),
]


@pytest.mark.parametrize("dims,slots,rank,n,order", BORDERS)
def test_forward_and_gradients_at_borders(dims, slots, rank, n, order):
    rng = np.random.default_rng(sum(dims) * 1000 + slots * 100 + rank + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, order)
    labels = rng.integers(0, dims[3], n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    logits, probs = forward(net, bank, x, s)
    want = tr.layers(params, flat, known(slots, s), 0.7, x, rank, dims)[4]
    tr.check(logits, want, "logits")
    tr.check(probs, tr.control(want, None, dims[3])[1], "probabilities")
    g, stats = grads(net, bank, x, labels, s)
    want, want_stats = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")


@pytest.mark.parametrize("rank", [5, 16, 24])
@pytest.mark.parametrize("n", [30, 700])
@pytest.mark.parametrize("off", [1, 2])
def test_inputs_at_any_address(rank, n, off):
    import torch
    dims, slots = (60, 96, 64, 12), 3
    rng = np.random.default_rng(rank + n + off)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 12, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    room = torch.zeros(n * 60 + off, device="cuda")
    room[off:] = dev(x).reshape(-1)
    ds, dl = dev(s), dev(labels)
    probs = torch.full((n * 12 + off + 1,), 7.0, device="cuda")
    net.forward_adapted_dev(bank, room.data_ptr() + 4 * off, ds.data_ptr(), n, probs_ptr=probs.data_ptr() + 4 * off)
    bank.zero_grad_dev()
    bank.accumulate_dev(net, room.data_ptr() + 4 * off, dl.data_ptr(), ds.data_ptr(), n)
    torch.cuda.synchronize()
    assert (probs[:off] == 7).all() and probs[-1] == 7
    want = tr.control(tr.layers(params, flat, known(slots, s), 0.7, x, rank, dims)[4], None, 12)[1]
    tr.check(probs[off:-1].reshape(n, 12).cpu().numpy(), want, "probabilities")
    got, _ = grads(net, bank, x, labels, s, zero=False)   # a second time on top of the first
    want, _ = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims)
    tr.check(got, tr.T(2 * want.v, 2 * want.e + tr.U * 2 * (np.abs(want.v) + want.e)), "gradient")


@pytest.mark.parametrize("dims,rank", [((60, 512, 64, 8), 16), ((60, 100, 70, 70), 20), ((60, 256, 2048, 3), 16)])
@pytest.mark.parametrize("n", [40, 700, 8200])
def test_values_that_are_none_stay_in_their_rows(dims, rank, n):
    """Rows of infinite or undefined inputs, and a slot of undefined factors, among others: these get what they get without them."""
    slots = 5
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    labels = rng.integers(0, dims[3], n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    logits, probs = forward(net, bank, x, s)
    bad = rng.integers(0, n, max(1, n // 30))
    y = x.copy()
    y[bad[::2]] = np.inf
    y[bad[1::2], 3] = np.nan
    sick = sz.Adapters(net, slots, rank, scale=0.7, init=np.where(np.arange(slots)[:, None] == 2, np.nan, flat).astype(np.float32))
    logits2, probs2 = forward(net, sick, y, s)
    fine = (s != 2) & ~np.isin(np.arange(n), bad)
    assert fine.any() and np.array_equal(logits[fine], logits2[fine]) and np.array_equal(probs[fine], probs2[fine])
    assert not np.isfinite(logits2[s == 2]).any()
    # the gradients of the slots that see none of those rows and factors
    clean = [k for k in range(slots) if k != 2]
    z = np.where(s == 3)[0]
    y = x.copy()
    y[z] = np.nan
    g, stats = grads(net, bank, x, labels, s)
    g2, stats2 = grads(net, sick, y, labels, s)
    for k in clean:
        if k != 3:
            assert np.array_equal(g[k], g2[k]) and np.array_equal(stats[k], stats2[k])


@pytest.mark.parametrize("rank", [8, 20])
def test_dropout_of_rows_in_tiles(rank):
    dims, slots, n = (60, 200, 32, 6), 3, 900
    rng = np.random.default_rng(rank)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 6, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    g, stats = grads(net, bank, x, labels, s, dropout=0.4, seed=5)
    xd = np.where(dropout_keep(5, n, 0.4), x, 0).astype(np.float32)
    want, want_stats = tr.train(params, flat, known(slots, s), 1.0, xd, labels, rank, dims)
    tr.check(stats, want_stats)
    tr.check(g, want)


def test_rows_of_zeros_do_not_count_in_tiles():
    dims, slots, rank, n = (60, 512, 64, 8), 4, 16, 1000
    rng = np.random.default_rng(3)
    params, flat, x = make(rng, dims, slots, rank, n)
    x[::3] = 0.0
    x[1::3] = 0.0
    x[1::3, 59] = -1e-30   # a single value, whatever its size
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(0, 8, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    _, stats = grads(net, bank, x, labels, s)
    live = x.any(axis=1)
    assert [int(v) for v in stats[:, 1]] == [int((live & (s == k)).sum()) for k in range(slots)]


def test_two_banks_of_one_net_on_two_streams():
    import torch
    dims, slots, n = (60, 512, 256, 16), 5, 4000
    rng = np.random.default_rng(21)
    params, flat, x = make(rng, dims, slots, 16, n)
    _, flat2, x2 = make(rng, dims, 3, 40, n)
    s, s2 = pick_slots(rng, n, slots, "mixed"), pick_slots(rng, n, 3, "mixed")
    net = sz.SimpleNeuralNet(*dims, init=params)
    banks = [sz.Adapters(net, slots, 16, init=flat), sz.Adapters(net, 3, 40, init=flat2)]
    data = [(dev(x), dev(s)), (dev(x2), dev(s2))]
    want = [forward(net, banks[0], x, s)[1], forward(net, banks[1], x2, s2)[1]]
    out = [torch.zeros(n, 16, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, (dx, ds), o, st in zip(banks, data, out, streams):
            net.forward_adapted_dev(b, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=o.data_ptr(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(out, want):
        assert np.array_equal(o.cpu().numpy(), w)


@pytest.mark.parametrize("classes", [1024, 51200, 51201])
def test_controls_where_a_row_no_longer_fits(classes):
    import torch
    rows, sets = 9, 3
    rng = np.random.default_rng(classes)
    z = rng.standard_normal((rows, classes)).astype(np.float32)
    c = host_controls(rng, sets, classes, rows)
    handle, keep = dev_controls(c)
    d = dev(z)
    out = torch.empty_like(d)
    sz.control_logits_dev(d.data_ptr(), rows, classes, handle, out.data_ptr(), probs=True)
    torch.cuda.synchronize()
    tr.check(out.cpu().numpy(), tr.control(tr.T(z), c, classes)[1], "probabilities")


@pytest.mark.parametrize("count", [4095, 4097, 9000])
def test_clip_a_group_of_very_many_tensors(count):
    import torch
    rng = np.random.default_rng(count)
    lens = rng.integers(0, 9, count)
    host = [rng.standard_normal(k).astype(np.float32) for k in lens]
    flat = dev(np.concatenate([np.concatenate([h, np.zeros(1, np.float32)]) for h in host]))
    at = np.concatenate([[0], np.cumsum(lens + 1)])[:-1]
    norm = float(np.sqrt(sum((h.astype(np.float64) ** 2).sum() for h in host)))
    norms = torch.zeros(1, device="cuda")
    clip = sz.GradClip([(flat.data_ptr() + 4 * int(a), int(k)) for a, k in zip(at, lens)])
    clip.run(0.25 * norm, norms.data_ptr())
    torch.cuda.synchronize()
    np.testing.assert_allclose(float(norms[0]), norm, rtol=2 * tr.U)
    got = flat.cpu().numpy()
    # the factor is formed in 64 bits: max_norm's rounding to 32 bits and the product's, at most (1 + U)^2 - 1 < 2.1 U
    for h, a, k in zip(host, at, lens):
        np.testing.assert_allclose(got[a:a + k], 0.25 * h.astype(np.float64), rtol=2.1 * tr.U, atol=0)
        assert got[a + k] == 0


def test_a_workspace_that_grows_call_by_call_stays_in_proportion():
    """Earlier workspaces are kept for the graphs that work in them; forty calls, each a little larger, must not keep forty of them."""
    import torch
    dims = (60, 512, 256, 16)
    rng = np.random.default_rng(2)
    params, flat, x = make(rng, dims, 2, 16, 16)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, 2, 16, init=flat)
    n = 4096 + 40 * 256
    dx, ds, out = torch.zeros(n, 60, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 16, device="cuda")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for k in range(41):
        net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), 4096 + 256 * k, probs_ptr=out.data_ptr())
    torch.cuda.synchronize()
    # 4096, 8192 and 16384 rows of 3.5 KB and three copies of the weights' tables: 110 MB; forty-one of them are 1.4 GB
    assert free - torch.cuda.mem_get_info()[0] < 300 << 20


def test_results_that_overlap_are_refused():
    import torch
    net = sz.SimpleNeuralNet(60, 32, 16, 4, seed=1)
    bank = sz.Adapters(net, 2, 3)
    n = 10
    x, s, o = torch.zeros(n * 60, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(2 * n * 4, device="cuda")
    a, b = o.data_ptr(), o.data_ptr() + 4 * 4 * n
    for kw in (dict(logits_ptr=a, probs_ptr=a), dict(logits_ptr=a, probs_ptr=b - 4), dict(logits_ptr=b - 4, probs_ptr=a),
               dict(probs_ptr=x.data_ptr()), dict(logits_ptr=x.data_ptr() + 4 * (60 * n - 1))):
        with pytest.raises(sz.StreamzError) as e:
            net.forward_adapted_dev(bank, x.data_ptr(), s.data_ptr(), n, **kw)
        assert e.value.code == -1 and "overlap" in str(e.value)
    net.forward_adapted_dev(bank, x.data_ptr(), s.data_ptr(), n, logits_ptr=a, probs_ptr=b)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dims", [(60, 64, 32, 8), (60, 64, 48, 100), (60, 64, 300, 300)])
@pytest.mark.parametrize("n", [1, 45, 700])
@pytest.mark.parametrize("asked", ["logits", "probs", "both"])
@pytest.mark.parametrize("sets", ["one", "by row"])
def test_forward_with_penalties_and_one_result_or_both(dims, n, asked, sets):
    import torch
    slots, rank, C = 3, 5, dims[3]
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    c = host_controls(rng, 4, C, n)
    c["counts"] = np.maximum(rng.integers(-5, 4, (4, C)), 0).astype(np.uint32)
    c["repetition"] = rng.uniform(0.6, 1.7, 4).astype(np.float32)
    c["presence"] = rng.uniform(-1, 1, 4).astype(np.float32)
    c["frequency"] = rng.uniform(-0.2, 0.2, 4).astype(np.float32)
    if sets == "one":
        c.pop("set_of_row")
    handle, keep = dev_controls(c)
    if sets == "one":
        c["set_of_row"] = np.zeros(n, np.int32)
    dx, ds = dev(x), dev(s)
    out = [torch.full((n + 1, C), 7.0, device="cuda") for _ in range(2)]
    net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, logits_ptr=out[0].data_ptr() if asked != "probs" else 0,
                            probs_ptr=out[1].data_ptr() if asked != "logits" else 0, controls=handle)
    torch.cuda.synchronize()
    want = tr.layers(params, flat, known(slots, s), 0.7, x, rank, dims)[4]
    if asked != "probs":
        tr.check(out[0][:n].cpu().numpy(), want, "logits")
    if asked != "logits":
        tr.check(out[1][:n].cpu().numpy(), tr.control(want, c, C)[1], "probabilities")
    assert (out[0][n] == 7).all() and (out[1][n] == 7).all()
    assert (out[0] == 7).all() or asked != "probs"
    assert (out[1] == 7).all() or asked != "logits"


@pytest.mark.parametrize("dims", [(60, 64, 32, 8), (60, 64, 48, 100), (60, 64, 300, 300)])
@pytest.mark.parametrize("n", [1, 60, 512, 513])
def test_votes_of_few_rows_and_of_tiles(dims, n):
    import torch
    slots, rank, groups, thr, C = 4, 3, 5, 0.01, dims[3]
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, group = pick_slots(rng, n, slots, "mixed"), rng.integers(-1, groups + 1, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    c = host_controls(rng, 3, C, n)
    handle, keep = dev_controls(c)
    _, probs = forward(net, bank, x, s, handle)
    dx, ds, dg = dev(x), dev(s), dev(group)
    for groups_of in (dg.data_ptr(), 0):
        counts = torch.full((groups, C), 3, dtype=torch.int64, device="cuda")
        net.vote_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, thr, counts.data_ptr(), groups=groups, group_of_row_ptr=groups_of, controls=handle)
        torch.cuda.synchronize()
        want = np.full((groups, C), 3, np.int64)
        for i in range(n):
            g = group[i] if groups_of else 0
            if 0 <= g < groups and probs[i].max() > 0 and probs[i].max() >= np.float32(thr):
                want[g, C - 1 - int(np.argmax(probs[i][::-1]))] += 1
        assert np.array_equal(counts.cpu().numpy(), want)


@pytest.mark.parametrize("dims,rank", [((60, 512, 64, 8), 16), ((60, 70, 50, 40), 20), ((60, 96, 72, 100), 7)])
def test_tiles_in_a_graph(dims, rank):
    """Other inputs and other slots at every replay, eager work between them."""
    import torch
    slots, n, C = 6, 1500, dims[3]
    rng = np.random.default_rng(sum(dims))
    params, flat, x = make(rng, dims, slots, rank, n)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    bank.reserve(n, training=True)
    c = host_controls(rng, 4, C, n)
    handle, keep = dev_controls(c)
    dx, ds, dl = dev(x), dev(pick_slots(rng, n, slots, "mixed")), dev(rng.integers(0, C, n).astype(np.int32))
    logits, probs = torch.zeros(n, C, device="cuda"), torch.zeros(n, C, device="cuda")
    from helpers import _DevView
    grad = torch.as_tensor(_DevView(bank.grad_ptr(), bank.grad_len()), device="cuda")

    def work(stream):
        net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, logits_ptr=logits.data_ptr(), probs_ptr=probs.data_ptr(), controls=handle,
                                stream=stream)
        bank.zero_grad_dev(stream)
        bank.accumulate_dev(net, dx.data_ptr(), dl.data_ptr(), ds.data_ptr(), n, controls=handle, stream=stream)
        bank.clip_grad_dev(0.01, 0, stream)
        bank.apply_grad_dev(0.1, stream)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        work(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        dx.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        ds.copy_(torch.from_numpy(pick_slots(rng, n, slots, "mixed")))
        start = [bank.get_params(k) for k in range(slots)]
        work(0)
        torch.cuda.synchronize()
        want = [t.clone() for t in (logits, probs, grad)]
        after = [bank.get_params(k) for k in range(slots)]
        for k in range(slots):
            bank.set_params(k, start[k])
        for t in (logits, probs, grad):
            t.fill_(-1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((logits, probs, grad), want):
            assert np.array_equal(a.cpu().numpy(), b.cpu().numpy(), equal_nan=True)
        for k in range(slots):
            assert all(np.array_equal(a, b) for a, b in zip(bank.get_params(k), after[k]))
