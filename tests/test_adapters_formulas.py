"""The plain forms that the GPU tests compare with, against differences of the loss, and the refusals that need no device."""
import ctypes as C

import numpy as np
import pytest

import streamz_amd as sz
import tracked as tr


def make(rng, dims, slots, rank, n):
    i, h1, h2, o = dims
    params = [rng.uniform(-1, 1, s) * (1.5 / np.sqrt(s[0]) if len(s) == 2 else 0.2) for s in ((i, h1), (h1,), (h1, h2), (h2,), (h2, o), (o,))]
    params = [p.astype(np.float32) for p in params]
    bank = (rng.uniform(-1, 1, (slots, rank * (h1 + 2 * h2 + o))) * 0.4).astype(np.float32)
    x = rng.standard_normal((n, i)).astype(np.float32)
    return params, bank, x


def test_plain_gradient_equals_differences_of_the_loss():
    rng = np.random.default_rng(1)
    dims, slots, rank, n = (5, 7, 6, 4), 3, 2, 9
    params, bank, x = make(rng, dims, slots, rank, n)
    bank = bank.astype(np.float64)
    sl = np.array([0, 1, -1, 0, 2, 5, 1, 1, 0])
    labels = np.array([0, 1, 2, 3, 0, 1, 3, -1, 2])
    x[6] = 0.0
    c = {"sets": 2, "set_of_row": np.array([0, 1, 0, 0, 1, 0, 1, 1, 0]), "bias": rng.standard_normal((2, 4)),
         "allow": np.array([[0b1111], [0b1011]], np.uint32)}
    grad, stats = tr.train(params, bank, sl, 0.5, x, labels, rank, dims, c)
    assert stats.v[:, 1].tolist() == [3, 1, 1]   # zero input, missing slot and label do not count

    def loss(b):
        return tr.train(params, b, sl, 0.5, x, labels, rank, dims, c)[1].v[:, 0].sum()

    step = 1e-5
    for s in range(slots):
        for k in range(bank.shape[1]):
            up, down = bank.copy(), bank.copy()
            up[s, k] += step
            down[s, k] -= step
            # central differences: third-derivative term of order step^2, rounding of order 1e-16 / step
            assert abs((loss(up) - loss(down)) / (2 * step) - grad.v[s, k]) < 1e-8


def test_a_label_outside_the_candidate_list_does_not_count():
    rng = np.random.default_rng(2)
    dims = (3, 4, 4, 3)
    params, bank, x = make(rng, dims, 1, 1, 2)
    c = {"sets": 1, "allow": np.array([[0b011]], np.uint32)}
    _, stats = tr.train(params, bank, np.zeros(2, int), 1.0, x, np.array([2, 1]), 1, dims, c)
    assert stats.v[0, 1] == 1


def test_control_of_a_row_without_candidates():
    z, p = tr.control(tr.T(np.array([[np.nan, np.inf, 1.0], [np.nan, 0.0, 1.0]])), {"sets": 2, "set_of_row": np.array([0, 1]),
                      "allow": np.array([[0], [0b110]], np.uint32)}, 3)
    assert np.isneginf(z.v[0]).all() and (p.v[0] == 0).all()
    assert p.v[1, 0] == 0 and abs(p.v[1].sum() - 1) < 1e-12


# ---- refusals: every one of them is decided before a device is looked for ------------------------------------

def refused(call, text):
    with pytest.raises(sz.StreamzError) as e:
        call()
    assert e.value.code == -1 and text in str(e.value)


A = 1 << 20   # addresses that nothing reads


@pytest.mark.parametrize("tensors,outputs,groups,text", [
    ([(A, 10), (A + 36, 10)], None, None, "overlap"),
    ([(A, 10), (A + 400, 10)], [A + 800, A + 836], None, "overlap"),
    ([(A, 10), (A + 400, 10)], [A + 800, A + 4], None, "read where"),
    ([(A, 10)], [A + 4], None, "read where"),
    ([(A + 2, 10)], None, None, "multiple of 4"),
    ([(0, 10)], None, None, "null"),
])
def test_clip_refuses_tensors_that_overlap_or_are_nowhere(tensors, outputs, groups, text):
    refused(lambda: sz.GradClip(tensors, outputs=outputs, groups=groups), text)


def test_clip_refuses_a_group_that_does_not_exist_and_no_groups():
    h = C.c_void_p()
    ptr, ln, gr = (C.c_void_p * 1)(A), np.array([4], np.uint64), np.array([1], np.uint32)
    L = sz.lib()
    assert L.szh_clip_create(ptr, None, ln.ctypes.data, gr.ctypes.data, 1, 1, None, C.byref(h)) == -1
    assert L.szh_clip_create(ptr, None, ln.ctypes.data, None, 1, 0, None, C.byref(h)) == -1
    assert L.szh_clip_create(ptr, None, ln.ctypes.data, None, 1, 1, None, None) == -1
    assert L.szh_clip_run_dev(None, 1.0, None, None) == -1
    assert L.szh_net_clip_grad_dev(None, 1.0, None, None) == -1


@pytest.mark.parametrize("kw,text", [
    (dict(controls=sz.LogitControls(sets=0)), "set"),
    (dict(controls=sz.LogitControls(sets=1, presence=A)), "counts"),
    (dict(ld_logits=15), "strides"),
    (dict(ld_out=15), "strides"),
    (dict(out_ptr=A + 64, ld_logits=16), "overlap"),
    (dict(out_ptr=A, ld_out=20), "overlap"),
    (dict(out_ptr=0), "null"),
    (dict(logits_ptr=0), "null"),
])
def test_controls_refuse(kw, text):
    kw = {**dict(logits_ptr=A, rows=4, classes=16, controls=None, out_ptr=A + (1 << 16)), **kw}
    refused(lambda: sz.control_logits_dev(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(rows=1 << 40, ld_logits=1 << 40), "too many"),     # (their product is 0 in 64 bits)
    (dict(rows=1 << 40, ld_out=1 << 30), "too many"),
    (dict(logits_ptr=A + 2), "multiple of 4"),
    (dict(out_ptr=A + (1 << 16) + 1), "multiple of 4"),
])
def test_controls_refuse_sizes_and_addresses_that_do_not_exist(kw, text):
    kw = {**dict(logits_ptr=A, rows=4, classes=16, controls=None, out_ptr=A + (1 << 16)), **kw}
    refused(lambda: sz.control_logits_dev(**kw), text)


def test_controls_refuse_an_unknown_result_and_take_empty_calls():
    L = sz.lib()
    assert L.szh_logits_control_dev(A, 4, 1, 4, None, 2, A + 4096, 4, None) == -1
    sz.control_logits_dev(0, 0, 16, None, 0)
    sz.control_logits_dev(0, 5, 0, None, 0)


def test_adapter_calls_refuse_missing_handles():
    L = sz.lib()
    h = C.c_void_p()
    assert L.szh_adapters_create(None, 1, 1, 1.0, None, 0, C.byref(h)) == -1
    assert L.szh_adapters_reserve(None, 1, 0) == -1
    assert L.szh_adapters_zero_grad_dev(None, None) == -1
    assert L.szh_adapters_clip_grad_dev(None, 1.0, None, None) == -1
    assert L.szh_adapters_apply_grad_dev(None, 1.0, None) == -1
    assert L.szh_adapters_get_params(None, 0, None) == -1
    assert L.szh_net_forward_adapted_dev(None, None, None, None, 0, None, None, None, None) == -1
    assert L.szh_net_vote_adapted_dev(None, None, None, None, 0, None, 0.5, None, 1, None, None) == -1
    assert L.szh_adapters_accumulate_dev(None, None, None, None, None, 0, None, 0.0, 0, None) == -1
    assert L.szh_adapters_param_count(None) == 0 and L.szh_adapters_grad_len(None) == 0 and not L.szh_adapters_grad_dev(None)
    L.szh_adapters_destroy(None)
    L.szh_clip_destroy(None)
