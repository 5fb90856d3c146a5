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
