"""Low-rank adapters and controls at values that are none, at the ends of the type's range, in workspaces that grow and in the kernels of
many classes, against the plain forms of tests/tracked.py."""
import numpy as np
import pytest

import streamz_amd as sz
import tracked as tr
from test_gpu_adapters import dev, dev_controls, forward, grads, host_controls, known, make, pick_slots

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,rank,n,mode", [
    ((60, 512, 256, 16), 16, 40, "f32"),      # row by row, back in the row's kernel
    ((60, 96, 300, 300), 7, 40, "f32"),       # row by row, the output layer and back as products of their own
    ((60, 512, 256, 16), 16, 700, "f32"),     # the output layer and back in one launch
    ((65, 100, 64, 8), 5, 700, "f32"),        # ... behind rows that are gathered first
    ((60, 100, 72, 40), 20, 700, "f32"),      # back in a launch of its own
    ((60, 96, 72, 100), 7, 700, "f32"),       # the output layer and back as products of their own
    ((60, 256, 256, 16), 16, 1100, "bf16x3"),
])
def test_rows_that_do_not_count_leave_no_trace(dims, rank, n, mode):
    """Rows without a label, with one that does not exist and with one off their candidate list: whatever they hold, infinities and NaN
    included, the gradients are those of the same call with ordinary values there, bit for bit."""
    slots, out = 4, dims[3]
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n, zero_rows=False)
    s, labels, row = pick_slots(rng, n, slots, "mixed"), rng.integers(0, out, n).astype(np.int32), np.arange(n)
    labels[row % 5 == 0], labels[row % 5 == 1] = -1, out
    c = {"sets": 2, "set_of_row": (row % 5 == 2).astype(np.int32), "allow": np.full((2, (out + 31) // 32), 0xffffffff, np.uint32)}
    labels[row % 5 == 2] = 3
    c["allow"][1, 0] &= ~np.uint32(1 << 3)
    y = x.copy()
    for k in range(3):
        at = row[row % 5 == k]
        y[at[::3]], y[at[1::3], 7], y[at[2::3]] = np.inf, np.nan, 3e38
    net = sz.SimpleNeuralNet(*dims, init=params)
    net.set_gemm(mode)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    handle, keep = dev_controls(c)
    g, stats = grads(net, bank, x, labels, s, handle)
    assert np.isfinite(g).all() and np.array_equal(g.any(axis=1), stats[:, 1] > 0)
    assert [int(v) for v in stats[:, 1]] == [int(((row % 5 > 2) & (s == k)).sum()) for k in range(slots)]
    g2, stats2 = grads(net, bank, y, labels, s, handle)
    assert np.array_equal(stats, stats2) and np.array_equal(g, g2)


@pytest.mark.parametrize("dims,rank", [((60, 512, 256, 16), 16), ((7, 33, 21, 5), 3), ((61, 37, 30, 70), 9), ((60, 64, 300, 300), 5)])
@pytest.mark.parametrize("n", [1, 9, 600])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("at", [0, -1])
def test_an_infinite_feature_is_carried_through(dims, rank, n, value, at):
    """With weights of one sign behind the first layer, an infinite feature makes hidden units 0 or inf, and tanh(inf) = 1: the logits
    are finite and known, in every kernel."""
    slots, (i, n1, n2, out) = 2, dims
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n, zero_rows=False)
    params[2], flat = np.abs(params[2]) + np.float32(0.01), np.abs(flat) + np.float32(0.01)
    assert (params[0][at] > 0).any() and (params[0][at] < 0).any()
    x[:, at] = value
    s = (np.arange(n) % 3 - 1).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    logits, probs = forward(net, bank, x, s)
    one = tr.T(np.ones((1, n2)))
    for k in range(-1, slots):
        want = tr.dot(one, tr.T(params[4]), rank + 1)
        if k >= 0:
            a3, b3 = tr.split(flat[k], tr.adapter_shapes(dims, rank))[2:]
            want = tr.add(want, tr.dot(tr.mul(tr.dot(one, tr.T(a3)), tr.T(np.float64(np.float32(0.7)))), tr.T(b3)))
        want = tr.add(want, tr.T(params[5]))
        rows = np.flatnonzero(s == k)
        want = tr.T(np.repeat(want.v, len(rows), 0), np.repeat(want.e, len(rows), 0))
        tr.check(logits[rows], want, "logits")
        tr.check(probs[rows], tr.control(want, None, out)[1], "probabilities")


def masks_around(rng, classes, sets):
    """About half of the classes, class 1 among them and class 0 not."""
    allow = rng.integers(0, 1 << 32, (sets, (classes + 31) // 32), dtype=np.uint32)
    allow[:, 0] = (allow[:, 0] & ~np.uint32(1)) | np.uint32(2)
    bits = (allow[:, np.arange(classes) // 32] >> (np.arange(classes) % 32).astype(np.uint32)) & 1
    return allow, bits.astype(bool)


@pytest.mark.parametrize("classes", [2, 7, 16, 33, 64, 100, 250, 500, 1000, 2000, 6000, 12000, 51000, 60001])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_class_off_the_list_has_no_probability_whatever_the_row_holds(classes, value, in_place):
    """A candidate's NaN or infinity makes every candidate's probability a NaN; the others stay at 0."""
    import torch
    rows = 6
    rng = np.random.default_rng(classes)
    z = rng.standard_normal((rows, classes)).astype(np.float32)
    allow, bits = masks_around(rng, classes, rows)
    z[::2, 1] = value
    z[1::2, 0] = value
    c = {"sets": rows, "allow": allow, "set_of_row": np.arange(rows, dtype=np.int32)}
    handle, keep = dev_controls(c)
    d = dev(z)
    out = d if in_place else torch.full_like(d, 7.0)
    sz.control_logits_dev(d.data_ptr(), rows, classes, handle, out.data_ptr(), probs=True)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert not got[~bits].any()
    assert np.isnan(got[::2][bits[::2]]).all() and np.isfinite(got[1::2]).all()


@pytest.mark.parametrize("dims,rank", [((60, 64, 32, 16), 4), ((60, 64, 48, 100), 20), ((60, 64, 32, 1200), 4), ((60, 64, 300, 300), 4)])
@pytest.mark.parametrize("n", [5, 600])
def test_a_class_off_the_list_has_no_probability_behind_the_adapters(dims, rank, n):
    slots, out = 2, dims[3]
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = (np.arange(n) % 2).astype(np.int32)
    flat[1, -1] = np.nan                     # the last class's factor: that logit of slot 1 alone is none
    allow, bits = masks_around(rng, out, 2)
    allow[:, -1] |= np.uint32(1 << ((out - 1) % 32))
    bits[:, -1] = True
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    c = {"sets": 2, "allow": allow, "set_of_row": s}
    handle, keep = dev_controls(c)
    logits, probs = forward(net, bank, x, s, handle)
    off = ~bits[s]
    assert np.isnan(logits[s == 1, -1]).all() and np.isfinite(logits[:, :-1]).all() and np.isfinite(logits[s == 0]).all()
    assert not probs[off].any() and np.isfinite(probs[s == 0]).all()
    assert np.isnan(probs[s == 1][bits[s[s == 1]]]).all()
    # the loss takes nothing from there either: the classes' own factors get no gradient
    labels = np.full(n, out - 1, np.int32)
    g, _ = grads(net, bank, x, labels, s, handle)
    b3 = g[:, rank * (dims[1] + 2 * dims[2]):].reshape(2, rank, out)
    for k in range(2):
        assert not b3[k][:, ~bits[k]].any()


def test_the_sum_of_a_row_of_very_many_classes():
    """1024 classes at the top and two million that are 2^-25 of them each: together 6 %, every one less than half a step of a sum
    that holds a top class."""
    import torch
    classes = (1 << 21) + 3
    low = np.float32(np.log(2.0 ** -25))
    z = np.full((2, classes), low, np.float32)
    z[0, :1024] = 0.0
    z[1, -1024:] = 0.0
    d = dev(z)
    out = torch.empty_like(d)
    sz.control_logits_dev(d.data_ptr(), 2, classes, None, out.data_ptr(), probs=True)
    torch.cuda.synchronize()
    e = np.exp(z.astype(np.float64))
    p = e / e.sum(axis=1, keepdims=True)
    # an exponential of at most 2 ulp and its exponent's rounding (18 U at most) in numerator and sum; a thread's sum in 64 bits, its rounding,
    # 6 + 15 additions across lanes and waves; the reciprocal and the product
    np.testing.assert_allclose(out.cpu().numpy(), p, rtol=(2 * (4 + 18) + 1 + 21 + 2) * tr.U, atol=0)


@pytest.mark.parametrize("classes", [16, 500, 3000])
@pytest.mark.parametrize("repetition", [2e-39, 1e-30, 1.3, 1e30, 1.6e38, 3.3e38])
def test_a_repetition_near_the_ends_of_the_range(classes, repetition):
    """z / repetition, that of the reciprocal and that of the product, also where the reciprocal of the repetition is no normal number."""
    import torch
    rng = np.random.default_rng(classes)
    z = (np.exp(rng.uniform(-80, 80, (4, classes))) * rng.choice([-1, 1], (4, classes))).astype(np.float32)
    rep = np.full(1, repetition, np.float32)
    c = {"sets": 1, "counts": np.ones((1, classes), np.uint32), "repetition": rep}
    handle, keep = dev_controls(c)
    d = dev(z)
    out = torch.empty_like(d)
    sz.control_logits_dev(d.data_ptr(), 4, classes, handle, out.data_ptr(), probs=False)
    torch.cuda.synchronize()
    wide = z.astype(np.float64)
    with np.errstate(over="ignore"):
        want = np.where(wide > 0, wide / np.float64(rep[0]), wide * np.float64(rep[0]))
    near = np.abs(np.abs(want) / 2.0 ** 128 - 1) < 4 * tr.U   # (these may round to infinity or not)
    inf = (np.abs(want) >= 2.0 ** 128) & ~near
    got = out.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isinf(got[~near]), inf[~near]) and (np.sign(got[inf]) == np.sign(want[inf])).all()
    # two roundings, (1 + U)^2 - 1, and that of a result below the normal numbers
    fine = ~inf & ~near
    np.testing.assert_array_less(np.abs(got[fine] - want[fine]), 2.001 * tr.U * np.abs(want[fine]) + 2.0 ** -150 + 1e-60)


@pytest.mark.parametrize("dims,rank,n", [((60, 64, 64, 16), 4, 16639), ((60, 128, 64, 16), 16, 13259), ((60, 30, 20, 70), 3, 13200), ((60, 64, 64, 16), 4, 33023)])
def test_gradients_of_just_fewer_rows_than_a_whole_step_of_chunks(dims, rank, n):
    """As many chunks of rows as a call can make beyond those that fill the chip."""
    slots = 3
    rng = np.random.default_rng(n)
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(-1, dims[3], n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    g, stats = grads(net, bank, x, labels, s)
    want, want_stats = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")


@pytest.mark.parametrize("dims,slots,rank,steps", [((60, 512, 256, 16), 2000, 16, (256, 700, 1300, 2100, 4000, 8192)),
                                                   ((60, 512, 256, 16), 3, 8, (300, 9000, 40000, 70000, 131072)),
                                                   ((60, 1024, 512, 100), 300, 32, (10, 500, 513, 3000, 6000))])
def test_a_training_workspace_that_grows_stays_in_proportion(dims, slots, rank, steps):
    """What a bank keeps after growing step by step, forward and training in turn, is at most twice what one that is reserved for the last
    step at once takes: the arrays of earlier steps together are no larger than the last ones, and what does not grow with the rows is there once."""
    import torch
    net = sz.SimpleNeuralNet(*dims, seed=1)
    banks = [sz.Adapters(net, slots, rank) for _ in range(2)]
    torch.cuda.synchronize()

    def taken(call):
        before = torch.cuda.mem_get_info()[0]
        call()
        torch.cuda.synchronize()
        return before - torch.cuda.mem_get_info()[0]

    def grow():
        for n in steps:
            banks[1].reserve(n)
            banks[1].reserve(n, training=True)

    once, grown = taken(lambda: banks[0].reserve(steps[-1], training=True)), taken(grow)
    # (each allocation is rounded up to 2 MiB: two for the rows of every step and four for the rest)
    assert once > 0 and grown <= 2 * once + (2 * len(steps) + 4) * (2 << 20)


def test_a_graph_keeps_its_arrays_while_the_workspace_grows():
    """Captured with the arrays of a small bank, replayed after larger calls have brought larger ones and worked in both."""
    import torch
    from helpers import _DevView
    dims, slots, rank, n = (60, 64, 64, 16), 5, 16, 300
    rng = np.random.default_rng(31)
    params, flat, x = make(rng, dims, slots, rank, 40000)
    s, labels = pick_slots(rng, 40000, slots, "mixed"), rng.integers(0, 16, 40000).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    want = grads(net, bank, x[:n], labels[:n], s[:n])
    dx, ds, dl = dev(x), dev(s), dev(labels)
    probs = torch.zeros(n, 16, device="cuda")
    net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=probs.data_ptr())
    torch.cuda.synchronize()
    want_probs = probs.clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        st = torch.cuda.current_stream().cuda_stream
        bank.zero_grad_dev(st)
        bank.accumulate_dev(net, dx.data_ptr(), dl.data_ptr(), ds.data_ptr(), n, stream=st)
        net.forward_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, probs_ptr=probs.data_ptr(), stream=st)
    P = bank.param_count()
    for more in (700, 5000, 40000):
        forward(net, bank, x[:more], s[:more])
        big = grads(net, bank, x[:more], labels[:more], s[:more])
        probs.zero_()
        graph.replay()
        torch.cuda.synchronize()
        g = torch.as_tensor(_DevView(bank.grad_ptr(), bank.grad_len()), device="cuda").cpu().numpy()
        assert np.array_equal(g[:slots * P].reshape(slots, P), want[0]) and np.array_equal(g[slots * P:].reshape(slots, 2), want[1])
        assert torch.equal(probs, want_probs)
        again = grads(net, bank, x[:more], labels[:more], s[:more])
        assert np.array_equal(big[0], again[0])


# 1024 classes and fewer: lanes of a wave a row; then a workgroup a row with 2, 4, 8, 16, 32 or 50 values a thread, then none kept
CLASSES = [1023, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769, 51200, 51201]


@pytest.mark.parametrize("classes", CLASSES)
def test_controls_of_many_classes(classes):
    import torch
    rows, sets = 7, 3
    rng = np.random.default_rng(classes)
    z = (3 * rng.standard_normal((rows, classes))).astype(np.float32)
    c = host_controls(rng, sets, classes, rows)
    c["counts"] = np.maximum(rng.integers(-5, 4, (sets, classes)), 0).astype(np.uint32)
    c["repetition"] = rng.uniform(0.6, 1.7, sets).astype(np.float32)
    c["presence"] = rng.uniform(-1, 1, sets).astype(np.float32)
    c["frequency"] = rng.uniform(-0.2, 0.2, sets).astype(np.float32)
    handle, keep = dev_controls(c)
    want_z, want_p = tr.control(tr.T(z), c, classes)
    for probs, want in ((True, want_p), (False, want_z)):
        d = dev(z)
        out = torch.full((rows + 1, classes), 7.0, device="cuda")
        sz.control_logits_dev(d.data_ptr(), rows, classes, handle, out.data_ptr(), probs=probs)
        sz.control_logits_dev(d.data_ptr(), rows, classes, handle, d.data_ptr(), probs=probs)
        torch.cuda.synchronize()
        tr.check(out[:rows].cpu().numpy(), want, "probabilities" if probs else "logits")
        assert torch.equal(d, out[:rows]) and (out[rows] == 7).all()


@pytest.mark.parametrize("classes", CLASSES)
def test_gradients_of_many_classes(classes):
    """Candidate lists, priors, labels that are missing, do not exist or are off the list."""
    dims, slots, rank, n = (60, 16, 8, classes), 3, 2, 261
    rng = np.random.default_rng(classes + 1)
    params, flat, x = make(rng, dims, slots, rank, n)
    s = pick_slots(rng, n, slots, "mixed")
    labels = rng.integers(0, classes, n).astype(np.int32)
    labels[::17], labels[5::17], labels[9::17], labels[12::17] = -1, classes, 0, classes - 1
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    c = host_controls(rng, 4, classes, n)
    handle, keep = dev_controls(c)
    g, stats = grads(net, bank, x, labels, s, handle)
    want, want_stats = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims, c)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")
    assert want_stats.v[:, 1].min() > 0
    again, stats2 = grads(net, bank, x, labels, s, handle)
    assert np.array_equal(g, again) and np.array_equal(stats, stats2)


@pytest.mark.parametrize("classes", CLASSES)
def test_votes_of_many_classes(classes):
    """The last of the largest, also where equal ones lie in other lanes, waves and steps of a thread."""
    import torch
    dims, slots, rank, n, groups, thr = (60, 16, 8, classes), 2, 2, 530, 3, 1e-7
    rng = np.random.default_rng(classes + 2)
    params, flat, x = make(rng, dims, slots, rank, n)
    # several classes with the same weights, which no other class can beat
    equal = np.unique(np.concatenate([rng.integers(0, classes, 5), [classes // 2, classes - 1 - classes // 3]]))
    params[4][:, equal] = params[4][:, equal[:1]]
    params[5][equal] = 30.0
    factors = flat.reshape(slots, -1)
    b3 = factors[:, rank * (16 + 2 * 8):].reshape(slots, rank, classes)
    b3[:, :, equal] = b3[:, :, equal[:1]]
    s, group = pick_slots(rng, n, slots, "mixed"), rng.integers(-1, groups + 1, n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=factors)
    c = {"sets": 3, "set_of_row": rng.integers(0, 3, n).astype(np.int32), "allow": np.full((3, (classes + 31) // 32), 0xffffffff, np.uint32)}
    last = equal[-1]
    c["allow"][1, last // 32] &= ~np.uint32(1 << (last % 32))   # the last of them is no candidate
    c["allow"][2] = 0
    handle, keep = dev_controls(c)
    dx, ds, dg = dev(x), dev(s), dev(group)
    counts = torch.ones(groups, classes, dtype=torch.int64, device="cuda")
    net.vote_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, thr, counts.data_ptr(), groups=groups, group_of_row_ptr=dg.data_ptr(), controls=handle)
    torch.cuda.synchronize()
    want = np.ones((groups, classes), np.int64)
    for i in range(n):
        if 0 <= group[i] < groups and c["set_of_row"][i] < 2:
            want[group[i], equal[-1 - c["set_of_row"][i]]] += 1
    assert np.array_equal(counts.cpu().numpy(), want)


@pytest.mark.parametrize("dims,rank,n", [((60, 256, 512, 16), 16, 1100), ((60, 512, 256, 100), 24, 1500), ((60, 256, 256, 20), 40, 1024)])
def test_gradients_in_split_bf16(dims, rank, n, monkeypatch):
    slots = 3
    rng = np.random.default_rng(sum(dims))
    params, flat, x = make(rng, dims, slots, rank, n)
    s, labels = pick_slots(rng, n, slots, "mixed"), rng.integers(-1, dims[3], n).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    net.set_gemm("bf16x3")
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    g, stats = grads(net, bank, x, labels, s)
    # products below 2^-24 of a term are dropped, one more rounding a product: every bound is linear in the rounding unit
    monkeypatch.setattr(tr, "U", 2 * tr.U)
    want, want_stats = tr.train(params, flat, known(slots, s), 0.7, x, labels, rank, dims)
    tr.check(stats, want_stats, "loss and live rows")
    tr.check(g, want, "gradient")
    again, _ = grads(net, bank, x, labels, s)
    assert np.array_equal(g, again)


@pytest.mark.parametrize("dims,rank", [((60, 512, 256, 16), 16), ((60, 40, 24, 70), 20), ((65, 64, 300, 300), 5)])
@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("at", [0, 31, -1])
def test_an_undefined_feature_leaves_no_hidden_unit(dims, rank, n, at):
    """v > 0 ? v : 0 of a NaN is 0 (lib.rs:882), in every kernel: the row's logits are those of hidden units of 0."""
    slots = 2
    rng = np.random.default_rng(sum(dims) + n)
    params, flat, x = make(rng, dims, slots, rank, n)
    x[:, at] = np.nan
    s = (np.arange(n) % 3 - 1).astype(np.int32)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, scale=0.7, init=flat)
    logits, _ = forward(net, bank, x, s)
    none = [np.zeros_like(p) for p in params[:2]] + params[2:]
    tr.check(logits, tr.layers(none, flat, known(slots, s), 0.7, np.zeros_like(x), rank, dims)[4], "logits")


@pytest.mark.parametrize("n", [60, 900])
def test_votes_in_a_graph(n):
    """Counts go on from replay to replay, beside eager calls of the same bank."""
    import torch
    dims, slots, rank, groups = (60, 64, 32, 8), 4, 3, 5
    rng = np.random.default_rng(n)
    params, flat, x = make(rng, dims, slots, rank, n)
    net = sz.SimpleNeuralNet(*dims, init=params)
    bank = sz.Adapters(net, slots, rank, init=flat)
    bank.reserve(n)
    dx, ds, dg = dev(x), dev(pick_slots(rng, n, slots, "mixed")), dev(rng.integers(-1, groups + 1, n).astype(np.int32))
    counts, eager = (torch.zeros(groups, 8, dtype=torch.int64, device="cuda") for _ in range(2))

    def work(out, stream):
        net.vote_adapted_dev(bank, dx.data_ptr(), ds.data_ptr(), n, 0.15, out.data_ptr(), groups=groups, group_of_row_ptr=dg.data_ptr(), stream=stream)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        work(counts, torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        dx.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
        ds.copy_(torch.from_numpy(pick_slots(rng, n, slots, "mixed")))
        torch.cuda.synchronize()
        work(eager, 0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(counts, eager) and int(counts.sum()) > 0
