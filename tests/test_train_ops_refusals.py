"""What the training operators refuse, on the CPU: every check comes before anything is enqueued."""
import ctypes as C
import math

import pytest
import torch

from litnicelm_b200 import plugin, training

BASE = 1 << 20  # an address that nothing dereferences
EINVAL = -1


def view(shape, dtype=0, strides=None, ptr=BASE, device=1):
    size = 2 if dtype == 2 else 4
    if strides is None:
        strides, at = [], size
        for d in reversed(shape):
            strides.insert(0, at)
            at *= d
    t = plugin.DevTensor(ptr, tuple(shape), tuple(strides), dtype, device).view()
    return t


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


def forward(lib, q=None, k=None, v=None, out=None, lse=BASE, options=True, work=BASE, size=1 << 30, **o):
    q = q or view((2, 8, 4, 16))
    k = k or view((2, 8, 2, 16))
    v = v or view((2, 8, 2, 16))
    out = out or view((2, 8, 4, 16), q.dtype)
    opts = training.AttentionOptions(o.get("scale", 0.25), 1, o.get("first", 0), o.get("window", 0), o.get("lengths"))
    return lib.litnice_b200_attention_forward(ref(q), ref(k), ref(v), ref(opts) if options else None, ref(out), lse, work,
                                              size, None)


@pytest.mark.parametrize("more,why", [
    (dict(q=view((2, 8, 64))), "q has rank 3"),
    (dict(q=view((2, 8, 4, 16), 1)), "neither f32 nor bfloat16"),
    (dict(q=view((2, 8, 4, 16), 2)), "k differs from q in type"),
    (dict(q=view((2, 8, 4, 16), device=0)), "not on the GPU"),
    (dict(q=view((2, 8, 4, 16), ptr=0)), "null data"),
    (dict(q=view((2, 8, 4, 16), ptr=BASE + 2)), "element boundary"),
    (dict(q=view((2, 0, 4, 16))), "extent of 0"),
    (dict(q=view((2, 8, 4, 16), strides=(2048, 256, 64, 3))), "no multiple of its element"),
    (dict(q=view((3, 8, 4, 16))), "number of streams"),
    (dict(q=view((2, 8, 4, 32))), "head dimension"),
    (dict(q=view((2, 8, 4, 132)), k=view((2, 8, 2, 132)), v=view((2, 8, 2, 132))), "more than 128"),
    (dict(q=view((2, 8, 3, 16))), "no multiple of the key heads"),
    (dict(v=view((2, 9, 2, 16))), "v differs from k"),
    (dict(v=view((2, 8, 2, 8))), "v differs from k"),
    (dict(out=view((2, 8, 4, 8))), "out differs from q"),
    (dict(out=view((2, 8, 4, 16), 2)), "out differs from q"),
    (dict(out=view((2, 8, 4, 16), strides=(0, 256, 64, 4))), "elements overlap"),
    (dict(out=view((2, 8, 4, 16), strides=(2048, 128, 64, 4))), "elements overlap"),
    (dict(lse=None), "lse is null"),
    (dict(lse=BASE + 1), "lse does not lie"),
    (dict(options=False), "null options"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(first=-1), "first"),
    (dict(first=(1 << 30) - 4), "first"),
    (dict(window=-1), "window"),
    (dict(lengths=BASE + 2), "lengths"),
    (dict(work=None), "null workspace"),
    (dict(work=BASE + 128), "256-byte"),
    (dict(size=0), "needed"),
], ids=lambda x: x if isinstance(x, str) else "")
def test_attention_forward_refuses(lib, more, why):
    assert forward(lib, **more) == EINVAL
    assert why in text(lib)


def test_attention_null_views(lib):
    o = training.AttentionOptions(1.0, 1, 0, 0, None)
    q = view((1, 1, 1, 4))
    for at in (0, 1, 2, 4):
        args = [ref(q), ref(q), ref(q), ref(o), ref(q), BASE, BASE, 1 << 30, None]
        args[at] = None
        assert lib.litnice_b200_attention_forward(*args) == EINVAL and "null view" in text(lib)
    assert lib.litnice_b200_attention_backward_workspace(None, None) == 0
    assert lib.litnice_b200_attention_forward_workspace(ref(q), ref(view((2, 1, 1, 4)))) == 0 and "streams" in text(lib)


def test_attention_backward_refuses(lib):
    q, k = view((2, 8, 4, 16)), view((2, 8, 2, 16))
    o = training.AttentionOptions(1.0, 1, 0, 0, None)
    need = lib.litnice_b200_attention_backward_workspace(ref(q), ref(k))
    assert need >= 2 * 8 * 4 * 4
    good = dict(dout=q, q=q, k=k, v=k, out=q, lse=BASE, o=o, dq=q, dk=k, dv=k, work=BASE, bytes=need)

    def call(**more):
        a = {**good, **more}
        return lib.litnice_b200_attention_backward(ref(a["dout"]), ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["out"]), a["lse"],
                                                   ref(a["o"]), ref(a["dq"]), ref(a["dk"]), ref(a["dv"]), a["work"], a["bytes"], None)

    for more, why in ((dict(work=None), "null workspace"), (dict(work=BASE + 4), "256-byte"), (dict(bytes=need - 1), "needed"),
                      (dict(dout=k), "dout differs"), (dict(out=k), "out differs"), (dict(dq=k), "dq differs"),
                      (dict(dk=q), "dk differs"), (dict(dv=view((2, 8, 2, 16), 2)), "dv differs"), (dict(lse=None), "lse"),
                      (dict(dk=view((2, 8, 2, 16), strides=(1024, 128, 0, 4))), "overlap"), (dict(dq=None), "null view")):
        assert call(**more) == EINVAL and why in text(lib), (more, text(lib))


def test_policy_loss_refuses(lib):
    z = view((4, 100))
    need = lib.litnice_b200_policy_loss_workspace(ref(z))
    good = dict(z=z, targets=BASE, old=BASE, adv=BASE, ref=None, weight=None, o=(1.0, 0.2, 0.2, 0.0), loss=BASE, logp=BASE, d=z,
                work=BASE, bytes=need)

    def call(**more):
        a = {**good, **more}
        o = training.PolicyOptions(*a["o"]) if a["o"] else None
        return lib.litnice_b200_policy_loss(ref(a["z"]), a["targets"], a["old"], a["adv"], a["ref"], a["weight"], ref(o), a["loss"],
                                            a["logp"], ref(a["d"]), a["work"], a["bytes"], None)

    for more, why in ((dict(z=view((4, 10, 10))), "rank"), (dict(z=view((4, 100), 1)), "neither"), (dict(z=None), "null view"),
                      (dict(z=view((4, 100), strides=(4, 16))), "columns of logits"),
                      (dict(targets=None), "targets"), (dict(old=None), "old_logp"), (dict(adv=None), "advantage"),
                      (dict(weight=BASE + 1), "weight"), (dict(o=None), "options"), (dict(o=(0.0, 0.2, 0.2, 0.0)), "temp"),
                      (dict(o=(-1.0, 0.2, 0.2, 0.0)), "temp"), (dict(o=(math.nan, 0.2, 0.2, 0.0)), "temp"),
                      (dict(o=(1e-45, 0.2, 0.2, 0.0)), "temp"), (dict(o=(1.0, 1.5, 0.2, 0.0)), "clip"),
                      (dict(o=(1.0, 0.2, -0.1, 0.0)), "clip"), (dict(o=(1.0, 0.2, math.nan, 0.0)), "clip"),
                      (dict(o=(1.0, 0.2, 0.2, math.inf)), "kl_weight"), (dict(o=(1.0, 0.2, 0.2, 0.1)), "ref_logp"),
                      (dict(loss=None), "loss"), (dict(logp=None), "logp"), (dict(d=view((4, 99))), "dlogits differs"),
                      (dict(d=view((4, 100), 2)), "dlogits differs"), (dict(d=view((4, 100), strides=(0, 4))), "overlap"),
                      (dict(d=view((4, 100), strides=(408, 4))), "another stride"),
                      (dict(d=view((4, 100), strides=(4, 16))), "columns of dlogits"),
                      (dict(work=None), "workspace"), (dict(bytes=need - 1), "needed")):
        assert call(**more) == EINVAL and why in text(lib), (more, text(lib))


def test_orthogonalise_and_muon_refuse(lib):
    x = view((3, 20, 30))
    need = lib.litnice_b200_orthogonalise_workspace(ref(x))
    assert need > 0

    def call(a=x, b=x, steps=5, work=BASE, size=need):
        return lib.litnice_b200_orthogonalise(ref(a), ref(b), steps, work, size, None)

    big = view((70000, 2, 2))
    for args, why in ((dict(a=view((20,))), "rank"), (dict(a=view((3, 20, 30), 2)), "not f32"), (dict(b=view((3, 30, 20))), "differs"),
                      (dict(b=view((3, 20, 30), strides=(0, 120, 4))), "overlap"), (dict(steps=-1), "steps"),
                      (dict(steps=101), "steps"), (dict(work=None), "workspace"), (dict(size=need - 1), "needed"),
                      (dict(a=big, b=big), "65535"), (dict(a=None), "null view")):
        assert call(**args) == EINVAL and why in text(lib), (args, text(lib))
    assert lib.litnice_b200_orthogonalise_workspace(ref(view((40000, 40000)))) == 0 and "40000" in text(lib)

    def muon(p=x, g=x, m=x, o=(0.1, 0.9, 0.0, 1, 5)):
        opts = training.MuonOptions(*o) if o else None
        return lib.litnice_b200_muon_step(ref(p), ref(g), ref(m), ref(opts), BASE, need, None)

    for args, why in ((dict(p=view((3, 30, 20))), "params differs"), (dict(m=view((1, 20, 30))), "momentum differs"),
                      (dict(o=None), "options"), (dict(o=(math.nan, 0.9, 0.0, 1, 5)), "not finite"),
                      (dict(o=(0.1, 0.9, 0.0, 1, -1)), "steps"), (dict(p=view((3, 20, 30), strides=(2400, 60, 4))), "overlap")):
        assert muon(**args) == EINVAL and why in text(lib), (args, text(lib))


def test_backend_stream_refuses(lib):
    st = C.c_void_p(5)
    assert lib.litnice_b200_backend_stream(None, C.byref(st)) == EINVAL and st.value is None
    assert lib.litnice_b200_backend_stream(None, None) == EINVAL


def test_python_layer_refuses():
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        training.attention_forward(x, x, x)
    with pytest.raises(TypeError, match="not a tensor"):
        training.muon_step(3, x, x, 0.1)
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        training.muon_step(x, x, x, 0.1)
    with pytest.raises(ValueError, match="not a CUDA tensor"):
        training.policy_loss(x[0, 0], x, x, x)


def test_results_on_other_tensors_are_refused(lib):
    """What begins where an argument does; slices of one buffer that begin elsewhere are taken."""
    at = [BASE * (i + 1) for i in range(9)]
    q, k, v = view((2, 8, 4, 16), ptr=at[0]), view((2, 8, 2, 16), ptr=at[1]), view((2, 8, 2, 16), ptr=at[2])
    for place, name in ((at[0], "q"), (at[1], "k"), (at[2], "v")):
        assert forward(lib, q=q, k=k, v=v, out=view((2, 8, 4, 16), ptr=place)) == EINVAL
        assert f"out lies on {name}" in text(lib)
    opts = training.AttentionOptions(0.25, 1, 0, 0, None)
    for moved, onto, why in ((2, 0, "dq lies on q"), (3, 1, "dk lies on k"), (4, 3, "dk lies on dv"), (2, 6, "dq lies on out"),
                             (4, 5, "dv lies on dout")):
        # q, k, dq, dk, dv, dout, out, v
        places = list(at)
        order = [0, 1, 2, 3, 4, 5, 6, 7]
        order[moved] = onto
        wide, narrow = (2, 8, 4, 16), (2, 8, 2, 16)
        shapes = (wide, narrow, wide, narrow, narrow, wide, wide, narrow)
        tq, tk, tdq, tdk, tdv, tdout, tout, tv = (view(s, ptr=places[o]) for s, o in zip(shapes, order))
        assert lib.litnice_b200_attention_backward(ref(tdout), ref(tq), ref(tk), ref(tv), ref(tout), BASE * 20, ref(opts), ref(tdq),
                                                   ref(tdk), ref(tdv), BASE * 30, 1 << 30, None) == EINVAL
        assert why in text(lib)
    mo = training.MuonOptions(0.1, 0.9, 0.0, 1, 5)
    for params, grads, momentum, why in ((0, 0, 1, "params lies on grads"), (0, 1, 0, "params lies on momentum"),
                                         (0, 1, 1, "momentum lies on grads")):
        views = [view((80, 96), ptr=at[i]) for i in (params, grads, momentum)]
        assert lib.litnice_b200_muon_step(*(ref(x) for x in views), ref(mo), BASE * 30, 1 << 30, None) == EINVAL
        assert why in text(lib)
