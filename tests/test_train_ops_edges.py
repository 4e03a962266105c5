"""Further calls that the training operators refuse, on the CPU: every check comes before anything is enqueued."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from litnicelm_b200 import plugin, training
from train_ops_calls import calls_with

BASE = 1 << 20  # an address that nothing dereferences
EINVAL, ECUDA = -1, -2


def view(shape, dtype=0, strides=None, ptr=BASE):
    size = 2 if dtype == 2 else 4
    if strides is None:
        strides, at = [], size
        for d in reversed(shape):
            strides.insert(0, at)
            at *= d
    return plugin.DevTensor(ptr, tuple(shape), tuple(strides), dtype, 1).view()


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(plugin.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return training._library()


def text(lib):
    return lib.litnice_b200_last_error(None).decode()


def ref(t):
    return None if t is None else C.addressof(t)


@pytest.mark.parametrize("shape,turned", [((5, 5, 20, 30), (2400, 12000, 120, 4)), ((4, 40, 40), (6400, 4, 160)),
                                          ((2, 3, 7, 80, 80), (591360, 197120, 28160, 352, 4))], ids=str)
def test_orthogonalise_in_place_wants_the_same_strides(lib, shape, turned):
    """One matrix of a call is written while another may still be read."""
    x, out = view(shape), view(shape, strides=turned)
    need = lib.litnice_b200_orthogonalise_workspace(ref(x))
    assert lib.litnice_b200_orthogonalise(ref(x), ref(out), 5, 64 * BASE, need, None) == EINVAL
    assert "out lies on x with another stride" in text(lib)


# every address of a call by itself, unless a case puts one onto another
AT = {name: BASE * (i + 1) for i, name in enumerate(
    ("q", "k", "v", "out", "lse", "lengths", "dout", "dq", "dk", "dv", "work", "logits", "targets", "old_logp", "advantage",
     "ref_logp", "weight", "loss", "logp", "dlogits", "x", "params", "grads", "momentum"))}
WIDE, NARROW = (2, 8, 4, 16), (2, 8, 2, 16)


def attention_forward(lib, at):
    o = training.AttentionOptions(0.25, 1, 0, 0, at["lengths"])
    tensors = [view(s, ptr=at[n]) for n, s in (("q", WIDE), ("k", NARROW), ("v", NARROW), ("out", WIDE))]
    q, k, v, out = (ref(t) for t in tensors)
    return lib.litnice_b200_attention_forward(q, k, v, ref(o), out, at["lse"], at["work"], 1 << 30, None)


def attention_backward(lib, at):
    o = training.AttentionOptions(0.25, 1, 0, 0, at["lengths"])
    tensors = [view(s, ptr=at[n]) for n, s in (("dout", WIDE), ("q", WIDE), ("k", NARROW), ("v", NARROW), ("out", WIDE), ("dq", WIDE),
                                               ("dk", NARROW), ("dv", NARROW))]
    dout, q, k, v, out, dq, dk, dv = (ref(t) for t in tensors)
    return lib.litnice_b200_attention_backward(dout, q, k, v, out, at["lse"], ref(o), dq, dk, dv, at["work"], 1 << 30, None)


def policy_loss(lib, at):
    o = training.PolicyOptions(1.0, 0.2, 0.2, 0.1)
    z, d = view((4, 100), ptr=at["logits"]), view((4, 100), ptr=at["dlogits"])
    return lib.litnice_b200_policy_loss(ref(z), at["targets"], at["old_logp"], at["advantage"], at["ref_logp"], at["weight"], ref(o),
                                        at["loss"], at["logp"], ref(d), at["work"], 1 << 30, None)


def orthogonalise(lib, at):
    x, out = view((80, 96), ptr=at["x"]), view((80, 96), ptr=at["out"])
    return lib.litnice_b200_orthogonalise(ref(x), ref(out), 5, at["work"], 1 << 30, None)


def muon_step(lib, at):
    o = training.MuonOptions(0.1, 0.9, 0.0, 1, 5)
    p, g, m = (view((80, 96), ptr=at[n]) for n in ("params", "grads", "momentum"))
    return lib.litnice_b200_muon_step(ref(p), ref(g), ref(m), ref(o), at["work"], 1 << 30, None)


@pytest.mark.parametrize("call,results,inputs", [
    (attention_forward, "out lse work", "q k v lengths"),
    (attention_backward, "dq dk dv work", "dout q k v out lse lengths"),
    (policy_loss, "loss logp dlogits work", "logits targets old_logp advantage ref_logp weight"),
    (orthogonalise, "work", "x out"), (muon_step, "work params momentum", "grads")], ids=lambda x: getattr(x, "__name__", ""))
def test_results_begin_where_nothing_else_does(lib, call, results, inputs):
    results, inputs = results.split(), inputs.split()
    pairs = [(r, x) for r in results for x in inputs] + [(a, b) for i, a in enumerate(results) for b in results[:i]]
    for one, other in pairs:
        if (one, other) == ("dlogits", "logits"):
            continue  # in place
        assert call(lib, {**AT, one: AT[other]}) == EINVAL, (one, other)
        names = [n.replace("work", "the workspace") for n in (one, other)]
        assert any(f"{a} lies on {b}" in text(lib) for a, b in (names, names[::-1])), (one, other, text(lib))


def test_too_many_blocks_are_refused_before_the_first_kernel(lib):
    """(Without a GPU the first kernel's launch would be an error of the runtime.)"""
    o = training.AttentionOptions(0.25, 1, 0, 0, None)
    for columns, m in ((4 * 8, 1), (4 * 9, 1), (4 * 8, 40)):  # rows that TMA can address, and not
        shape, keys = (1 << 21, 1, 1 << 10, 8), (1 << 21, m, 1 << 10, 8)
        q = [view(shape, 2, (columns << 10, columns << 10, columns, 2), BASE * (i + 1)) for i in range(4)]
        k = [view(keys, 2, (m * columns << 10, columns << 10, columns, 2), BASE * (i + 5)) for i in range(4)]
        assert lib.litnice_b200_attention_backward(ref(q[0]), ref(q[1]), ref(k[0]), ref(k[1]), ref(q[2]), 9 * BASE, ref(o), ref(q[3]),
                                                   ref(k[2]), ref(k[3]), 10 * BASE, 1 << 62, None) == EINVAL
        assert "too many rows, heads and streams" in text(lib)
    x, y, z = (view((60000, 8192, 1 << 22), ptr=BASE * (i + 1)) for i in range(3))
    assert lib.litnice_b200_orthogonalise_workspace(ref(x)) == 0 and "too many matrices" in text(lib)
    assert lib.litnice_b200_orthogonalise(ref(x), ref(y), 5, 4 * BASE, 1 << 62, None) == EINVAL and "too many matrices" in text(lib)
    mo = training.MuonOptions(0.1, 0.9, 0.0, 1, 5)
    assert lib.litnice_b200_muon_step(ref(x), ref(y), ref(z), ref(mo), 4 * BASE, 1 << 62, None) == EINVAL
    assert "too many matrices" in text(lib)


@pytest.mark.parametrize("stride", [1 << 51, -(1 << 51), -(1 << 63)])
def test_impossible_strides(lib, stride):
    at = [BASE * (i + 1) for i in range(6)]
    q, k, v, out = (view(WIDE if i % 3 == 0 else NARROW, ptr=at[i]) for i in range(4))
    o = training.AttentionOptions(0.25, 1, 0, 0, None)
    bad = view(WIDE, strides=(stride, 256, 64, 4), ptr=at[0])
    assert lib.litnice_b200_attention_forward(ref(bad), ref(k), ref(v), ref(o), ref(out), at[4], at[5], 1 << 30, None) == EINVAL
    assert "q has an impossible stride" in text(lib)
    assert lib.litnice_b200_attention_forward(ref(q), ref(k), ref(v), ref(o), ref(bad), at[4], at[5], 1 << 30, None) == EINVAL
    assert "out has an impossible stride" in text(lib)


@pytest.mark.parametrize("shape", [(1, 4, 2, 8), (2, 8)])
def test_views_of_negated_values_are_refused(shape):
    x = torch.zeros(*shape, dtype=torch.complex64).conj().imag
    assert x.dtype == torch.float32 and x.is_neg()
    for call in calls_with(x, x):
        with pytest.raises(ValueError, match="negated"):
            call()


@pytest.mark.parametrize("shape", [(1, 4, 2, 8), (2, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangents_are_refused(shape, dtype):
    x = torch.zeros(*shape, dtype=dtype)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls_with(dual, dual):
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls_with(x, x):  # those without one get as far as the device
            with pytest.raises(ValueError, match="not a CUDA tensor"):
                call()


@pytest.mark.parametrize("steps", [-1, 101, (1 << 32) + 5, -(1 << 32)])
def test_steps_beyond_32_bits(steps):
    """(An integer of ctypes takes the lowest bits of what it is given.)"""
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="steps is out of range"):
        training.orthogonalise(x, steps=steps)
    with pytest.raises(ValueError, match="steps is out of range"):
        training.muon_step(x, x, x, 0.1, steps=steps)
