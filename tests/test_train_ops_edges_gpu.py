"""The training operators where calls come close to what they were not made for, through litnicelm_b200.training."""
import math
import os
import subprocess
import sys
import threading

import pytest
import torch
from torch.autograd import forward_ad

from litnicelm_b200 import training
from train_ops_calls import calls_with
from train_ops_util import check, loss_reference, seen_keys

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- two calls at once from two host threads --------------------------------------------------------------------------------------


def at_once(*calls):
    """Each call from its own thread and stream, all starting together; what they return."""
    gate, results = threading.Barrier(len(calls)), [None] * len(calls)

    def run(i):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        try:
            with torch.cuda.stream(stream):
                gate.wait()
                results[i] = calls[i]()
        except Exception as e:  # for the assertion in the main thread
            results[i] = e
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return results


def test_small_matrices_of_two_sizes_from_two_threads():
    """Each size wants its own amount of shared memory of one kernel."""
    g = gen(1)
    sets = [rand(g, *shape) for shape in ((64, 64), (64, 4096), (20, 1000))]
    alone = [training.orthogonalise(x) for x in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = at_once(*(lambda x=x: [training.orthogonalise(x) for _ in range(400)] for x in sets))
        for a, results in zip(alone, got):
            assert not isinstance(results, Exception), results
            assert all(torch.equal(a, b) for b in results)


# ---- weights that cancel ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [96, 5001, 32000, 70000])
def test_policy_loss_weights_that_cancel(dtype, vocab):
    """Weights without a sum, all zero or not, give loss 0 and gradients of 0; the log probabilities are those of any weight."""
    g = gen(2)
    logits = rand(g, 6, vocab, dtype=dtype)
    targets = torch.randint(0, vocab, (6,), generator=g, device="cuda", dtype=torch.int32)
    old, adv, ref = (rand(g, 6) - 9 for _ in range(3))
    more = dict(ref_logp=ref, kl_weight=0.1)
    want = training.policy_loss(logits, targets, old, adv, **more)[1]
    weight = torch.tensor([1.0, -2, 0, 3, -1, -1], device="cuda")
    loss, logp, d = training.policy_loss(logits, targets, old, adv, weight=weight, **more)
    assert float(loss) == 0 and bool((d == 0).all())
    assert torch.equal(logp, torch.where(weight != 0, want, torch.zeros_like(want)))


# ---- rows that see no key ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 33])
@pytest.mark.parametrize("m,lengths,opts", [
    (300, [100, 33, 0, 256], dict(window=40)), (300, [130, 1, 200, 255], dict(window=3)), (90, None, dict(window=40)),
    (300, [77, 128, 0, 290], dict(window=100, causal=False)), (200, [60, 150, 5, 0], dict(first=30, window=25)),
    (100, None, dict(first=400, window=7))], ids=str)
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_rows_that_see_no_key_reach_nothing(dtype, dim, m, lengths, opts, fill):
    """Whatever their queries and upstream gradients hold."""
    g = gen(3)
    streams, n, heads = 4, 300, 4
    q, dout = (rand(g, streams, n, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (rand(g, streams, m, 2, dim, dtype=dtype) for _ in range(2))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    seen = seen_keys(n, m, opts.get("causal", True), opts.get("first", 0), opts["window"], lens, streams, "cuda")
    empty = ~seen.any(3).expand(streams, 1, n)[:, 0]
    assert bool(empty.any())
    results = []
    for x in (0.0, fill):
        q[empty], dout[empty] = x, x
        out, lse = training.attention_forward(q, k, v, lengths=lens, **opts)
        results.append((out, lse, *training.attention_backward(dout, q, k, v, out, lse, lengths=lens, **opts)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    out, lse, dq = results[1][:3]
    assert bool((out[empty] == 0).all()) and bool((dq[empty] == 0).all())
    assert bool((lse.transpose(1, 2)[empty] == -math.inf).all())


# ---- scores far from zero ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,n", [(64, 100), (64, 300), (128, 150), (33, 90)])
@pytest.mark.parametrize("size", [1e4, 1e10, 1e16])
def test_forward_all_scores_far_below_zero(dtype, dim, n, size, factor=-1.0):
    """Equal scores, however low: the mean of the values. The weights are 1 exactly, their sum a whole number; a product over n keys is
    off by 2 n u of the sum of magnitudes, its rounding by half a step."""
    g = gen(4)
    q = torch.full((1, n, 2, dim), size, device="cuda").to(dtype)
    k, v = (factor * q), rand(g, 1, n, 2, dim, dtype=dtype)
    out, lse = training.attention_forward(q, k, v)
    count = torch.arange(1, n + 1, device="cuda", dtype=torch.float64)
    V = v.double()
    want, mean = V.cumsum(1) / count[:, None, None], V.abs().cumsum(1) / count[:, None, None]
    h = torch.finfo(dtype).eps / 2
    bound = (2 * n + 8) * 2.0 ** -24 * mean
    assert bool(((out.double() - want).abs() <= bound + h * (want.abs() + bound)).all())
    score = factor * float(q.flatten()[0]) ** 2 * dim * dim ** -0.5
    # a sum of dim equal products and the scale; the log of the count
    assert bool(((lse.double() - (score + count.log())).abs() <= (2 * dim + 16) * 2.0 ** -24 * (abs(score) + count.log() + 1)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,n", [(64, 100), (64, 300), (128, 150), (33, 90)])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e12])
def test_forward_weight_on_one_key(dtype, dim, n, size):
    """Scores whose largest is ahead of the others by more than they are off by: the row is that key's value, rounded once more at most."""
    g = gen(5)
    q, k = ((rand(g, 1, n, 2, dim) * size).to(dtype) for _ in range(2))
    v = rand(g, 1, n, 2, dim, dtype=dtype)
    out, lse = training.attention_forward(q, k, v)
    Q, K = (x.double().transpose(1, 2) for x in (q, k))
    s = Q @ K.mT * dim ** -0.5
    off = ((dim + 8) * 2 * 2.0 ** -24 * (Q.abs() @ K.abs().mT) * dim ** -0.5).amax(3)
    s = torch.where(seen_keys(n, n, True, 0, 0, None, 1, "cuda"), s, torch.full_like(s, -math.inf))
    top = s.topk(2, 3)
    alone = top.values[..., 0] - top.values[..., 1] > 2 * off + 60  # the others' weights are below 2^-80
    assert bool(alone[:, :, 1:].any())
    at = top.indices[..., 0]
    want = v.transpose(1, 2).gather(2, at[..., None].expand(-1, -1, -1, dim)).double()
    got = out.transpose(1, 2).double()
    # the weight and the sum that divides by it are the same number, in bfloat16's product rounded once
    h = (torch.finfo(dtype).eps if dtype == BF16 else 8 * 2.0 ** -24)
    assert bool(((got - want).abs() <= h * want.abs() + 1e-20)[alone].all())
    assert bool(((lse.double() - top.values[..., 0]).abs() <= off + 8 * 2.0 ** -24 * top.values[..., 0].abs() + 1e-6)[alone].all())


# ---- results in memory that the caller gives --------------------------------------------------------------------------------------


def test_given_results_count_as_changed():
    g = gen(6)
    q, k, v = (rand(g, 1, 20, 2, 16) for _ in range(3))
    given = {n: torch.empty_like(q) for n in ("out", "dq", "dk", "dv")}
    z, x, u = rand(g, 4, 30), rand(g, 8, 12), rand(g, 8, 12)
    targets, old, adv = torch.zeros(4, dtype=torch.int32, device="cuda"), rand(g, 4), rand(g, 4)
    p, m = rand(g, 8, 12), rand(g, 8, 12)
    before = {n: t._version for n, t in {**given, "z": z, "u": u, "x": x, "p": p, "m": m, "q": q, "k": k, "v": v}.items()}
    out, lse = training.attention_forward(q, k, v, out=given["out"])
    training.attention_backward(q, q, k, v, out, lse, dq=given["dq"], dv=given["dv"])
    training.policy_loss(z, targets, old, adv, dlogits=z)
    training.orthogonalise(x, out=u)
    training.muon_step(p, x, m, 0.1)
    after = {n: t._version for n, t in {**given, "z": z, "u": u, "x": x, "p": p, "m": m, "q": q, "k": k, "v": v}.items()}
    changed = {n for n in before if after[n] != before[n]}
    assert changed == {"out", "dq", "dv", "z", "u", "p", "m"}


def test_autograd_sees_that_a_step_changed_what_it_saved():
    g = gen(7)
    p = rand(g, 8, 12).requires_grad_()
    loss = (p * p).sum()
    with torch.no_grad():
        training.muon_step(p, rand(g, 8, 12), torch.zeros(8, 12, device="cuda"), 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # tensors without a version
        a, b, c = (torch.ones(8, 12, device="cuda") for _ in range(3))
        training.muon_step(a, b, c, 0.1)
        assert bool((c == 1.95).all())


# ---- tensors that are more than their memory ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [(1, 4, 2, 8), (2, 8)])
def test_memory_that_is_not_all_of_a_tensor(shape):
    """In any place of a call: refused, and nothing written."""
    other = rand(gen(8), *shape)
    vectors = torch.zeros(2, dtype=torch.complex64, device="cuda").conj().imag
    if len(shape) == 2:
        ids, n = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
        for more in (dict(old_logp=vectors), dict(advantage=vectors), dict(ref_logp=vectors), dict(weight=vectors)):
            with pytest.raises(ValueError, match="negated"):
                training.policy_loss(other, ids, **{"old_logp": n, "advantage": n, **more})
    x = torch.ones(*shape, dtype=torch.complex64, device="cuda").conj().imag
    for call in calls_with(x, other):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert bool((x == 0).all())
    with forward_ad.dual_level():
        y = torch.ones(*shape, device="cuda")
        for call in calls_with(forward_ad.make_dual(y, torch.ones_like(y)), other):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert bool((y == 1).all())


@pytest.mark.parametrize("shape", [(1, 4, 2, 8), (2, 8)])
def test_gradients_that_autograd_would_want(shape):
    other, x = rand(gen(9), *shape), rand(gen(10), *shape).requires_grad_()
    for call in calls_with(x, other):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


# ---- policy loss: rows of every length and boundary ----------------------------------------------------------------------------------


def wide_loss(dtype, rows, vocab, ld, dld, in_place):
    """Rows of logits `ld` elements apart and of the gradient `dld`; the last column is one row's target, the first another's. What lies
    between the gradient's rows stays."""
    g = gen(vocab + ld)
    buffer = rand(g, rows, ld, dtype=dtype) * 2
    logits = buffer[:, :vocab]
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    targets[0], targets[1] = vocab - 1, 0
    now = torch.log_softmax(logits.double(), 1).gather(1, targets.long()[:, None])[:, 0]
    old, refp = ((now + s * rand(g, rows).double()).float() for s in (0.3, 0.4))
    adv, weight = rand(g, rows), torch.ones(rows, device="cuda")
    weight[2] = 0
    ref = loss_reference(logits, targets, old, adv, ref=refp, weight=weight, kl=0.1)
    out = buffer if in_place else torch.full((rows, dld), 7.0, dtype=dtype, device="cuda")
    before = out[:, vocab:].clone()
    loss, logp, d = training.policy_loss(logits, targets, old, adv, ref_logp=refp, weight=weight, kl_weight=0.1, dlogits=out[:, :vocab])
    check("loss", loss, ref["loss"])
    check("logp", logp, ref["logp"])
    keep = ~ref["near"]
    check("dlogits", d[keep], tuple(x[keep] for x in ref["dlogits"]))
    assert torch.equal(out[:, vocab:], before)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1021, 1025, 8191, 8193, 12001, 16383, 16385, 20003, 32001, 32767, 32769])
def test_policy_loss_rows_off_16_bytes(dtype, vocab):
    wide_loss(dtype, 5, vocab, vocab, vocab, False)
    wide_loss(dtype, 5, vocab, vocab + 2, (vocab + 15) // 8 * 8, False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1021, 8193, 10001, 16389, 32001, 32767, 32768, 40001])
@pytest.mark.parametrize("rows", [5, 300])
def test_policy_loss_rows_with_a_tail(dtype, vocab, rows):
    """On 16-byte boundaries, of columns that vectors do not divide."""
    ld = (vocab + 15) // 8 * 8
    wide_loss(dtype, rows, vocab, ld, vocab, False)
    wide_loss(dtype, rows, vocab, ld, ld + 8, False)
    wide_loss(dtype, rows, vocab, ld, ld, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [90, 8193, 32001, 50001])
def test_policy_loss_without_gradient(dtype, vocab):
    g = gen(12)
    for ld in (vocab, (vocab + 7) // 8 * 8):
        logits = rand(g, 7, ld, dtype=dtype)[:, :vocab]
        targets = torch.randint(0, vocab, (7,), generator=g, device="cuda", dtype=torch.int32)
        old, adv = -9 + rand(g, 7), rand(g, 7)
        a = training.policy_loss(logits, targets, old, adv, gradient=False)
        b = training.policy_loss(logits, targets, old, adv)
        assert a[2] is None and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- several operators at once, captured and not --------------------------------------------------------------------------------------


def passes():
    """Calls that share kernels in other forms: types, head dimensions, sizes of matrices, lengths of rows."""
    g = gen(20)

    def attention(dtype, n, dim, **more):
        q, dout = (rand(g, 3, n, 4, dim, dtype=dtype) for _ in range(2))
        k, v = (rand(g, 3, n, 2, dim, dtype=dtype) for _ in range(2))
        lens = torch.tensor([n, n // 2, 0], dtype=torch.int32, device="cuda")

        def run():
            out, lse = training.attention_forward(q, k, v, lengths=lens, **more)
            return (out, lse, *training.attention_backward(dout, q, k, v, out, lse, lengths=lens, **more))
        return run

    def loss(dtype, rows, vocab):
        z = rand(g, rows, vocab, dtype=dtype)
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        old, adv, w = -9 + rand(g, rows), rand(g, rows), (rand(g, rows) > 0).float()
        return lambda: training.policy_loss(z, t, old, adv, weight=w)

    def step(*shape):
        p, d, m = (rand(g, *shape) for _ in range(3))

        def run():
            a, b = p.clone(), m.clone()
            training.muon_step(a, d, b, 0.02)
            return a, b
        return run

    return [attention(F32, 200, 64), attention(F32, 150, 128, window=30), attention(BF16, 300, 64), attention(BF16, 300, 128),
            attention(BF16, 120, 33), loss(F32, 300, 9000), loss(BF16, 40, 32000), loss(F32, 50, 40000), step(2, 64, 256), step(5, 300),
            step(3, 200, 150), step(1024, 300)]


def test_operators_from_several_threads():
    calls = passes()
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        got = at_once(*(lambda call=call: [call() for _ in range(20)] for call in calls))
        for a, results in zip(alone, got):
            assert not isinstance(results, Exception), results
            for b in results:
                assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_operators_captured_beside_eager_ones():
    """One graph of all, replayed while the same calls run on another stream."""
    calls = passes()
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call() for call in calls]
    side = torch.cuda.Stream()
    for _ in range(5):
        for results in captured:
            for x in results:
                x.fill_(float("nan"))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            eager = [call() for call in calls]
        torch.cuda.synchronize()
        for a, b, c in zip(alone, captured, eager):
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    del captured, graph  # before the process ends


# ---- keys that no row sees ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 33])
@pytest.mark.parametrize("n,m,lengths,opts", [
    (100, 300, None, dict()), (300, 500, None, dict(window=50)), (1, 200, None, dict(first=70)), (130, 400, [400, 200, 100, 0], dict(first=60)),
    (70, 200, None, dict(first=100, window=10)), (200, 300, [250, 300, 1, 190], dict(window=1))], ids=str)
@pytest.mark.parametrize("fill", [math.nan, -math.inf])
def test_keys_that_no_row_sees_reach_nothing(dtype, dim, n, m, lengths, opts, fill):
    """The unused end of a cache, and what lies before every row's window, may hold anything."""
    g = gen(13)
    streams, heads = 4, 4
    q, dout = (rand(g, streams, n, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (rand(g, streams, m, 2, dim, dtype=dtype) for _ in range(2))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    seen = seen_keys(n, m, True, opts.get("first", 0), opts.get("window", 0), lens, streams, "cuda")
    unseen = ~seen.any(2).expand(streams, 1, m)[:, 0]
    assert bool(unseen.any())
    results = []
    for x in (0.0, fill):
        k[unseen], v[unseen] = x, x
        out, lse = training.attention_forward(q, k, v, lengths=lens, **opts)
        results.append((out, lse, *training.attention_backward(dout, q, k, v, out, lse, lengths=lens, **opts)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert bool((results[1][3][unseen] == 0).all()) and bool((results[1][4][unseen] == 0).all())


# ---- far apart, and in any order ----------------------------------------------------------------------------------------------------


def far(rows, *shape, dtype=F32):
    """`rows` blocks of zeros, each as far from the next as 2^31 elements and some leave them."""
    size = math.prod(shape)
    step = ((1 << 31) // (rows - 1) + 8192) // 8 * 8
    buffer = torch.empty((rows - 1) * step + size, dtype=dtype, device="cuda")
    strides = [math.prod(shape[i + 1:]) for i in range(len(shape))]
    out = torch.as_strided(buffer, (rows, *shape), (step, *strides))
    out.zero_()
    return out


@pytest.mark.parametrize("dtype,dim", [(F32, 40), (BF16, 64), (BF16, 128), (BF16, 33)])
def test_attention_streams_far_apart(dtype, dim):
    g = gen(14)
    near = [rand(g, 2, 140, h, dim, dtype=dtype) for h in (4, 2, 2, 4)]
    out, lse = training.attention_forward(*near[:3])
    want = (out, *training.attention_backward(near[3], *near[:3], out, lse))
    for place in range(4):  # one operand at a time
        x = far(2, 140, near[place].shape[2], dim, dtype=dtype)
        x.copy_(near[place])
        args = [x if i == place else t for i, t in enumerate(near)]
        result = torch.empty_like(out)
        o, s = training.attention_forward(*args[:3], out=result)
        got = (o, *training.attention_backward(args[3], *args[:3], o, s))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        del x, args
    for place in range(4):  # and one result
        x = far(2, 140, want[place].shape[2], dim, dtype=dtype)
        if place == 0:
            training.attention_forward(*near[:3], out=x)
        else:
            training.attention_backward(near[3], *near[:3], out, lse, **{("dq", "dk", "dv")[place - 1]: x})
        assert torch.equal(x, want[place])
        del x


@pytest.mark.parametrize("vocab", [96, 5000, 20001, 32000, 40000])
def test_policy_loss_rows_far_apart(vocab):
    g = gen(15)
    z = rand(g, 4, vocab, dtype=BF16)
    targets = torch.randint(0, vocab, (4,), generator=g, device="cuda", dtype=torch.int32)
    old, adv = -9 + rand(g, 4), rand(g, 4)
    want = training.policy_loss(z, targets, old, adv)
    x = far(4, vocab, dtype=BF16)
    x.copy_(z)
    got = training.policy_loss(x, targets, old, adv)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    training.policy_loss(x, targets, old, adv, dlogits=x)
    assert torch.equal(x, want[2])


@pytest.mark.parametrize("shape", [(40, 70), (200, 300), (300, 200)])
def test_matrices_far_apart_and_turned(shape):
    """Weights, gradients and momentum each in their own order of memory."""
    g = gen(16)
    p, d, m = (rand(g, 2, *shape) for _ in range(3))
    a, b = p.clone(), m.clone()
    training.muon_step(a, d, b, 0.03, weight_decay=0.1)
    for place in range(3):
        for form in ("far", "turned", "apart"):
            if form == "far":
                x = far(2, *shape)
            elif form == "turned":
                x = torch.empty(2, shape[1], shape[0], device="cuda").mT
            else:
                x = torch.empty(2, shape[0], 2, shape[1], 3, device="cuda")[:, :, 1, :, 1]
            args = [p.clone(), d, m.clone()]
            x.copy_(args[place])
            args[place] = x
            training.muon_step(*args[:2], args[2], 0.03, weight_decay=0.1)
            assert torch.equal(args[0], a) and torch.equal(args[2], b) and torch.equal(args[1], d)
            del x, args
    e = torch.zeros(1, *shape, device="cuda").expand(2, -1, -1)  # a broadcast gradient
    p2, m2 = p.clone(), m.clone()
    training.muon_step(p2, e, m2, 0.03)
    p3, m3 = p.clone(), m.clone()
    training.muon_step(p3, e.contiguous(), m3, 0.03)
    assert torch.equal(p2, p3) and torch.equal(m2, m3)


def test_first_calls_of_a_process_inside_a_capture():
    code = """
import torch
from litnicelm_b200 import training
g = torch.Generator(device="cuda").manual_seed(1)
x = [torch.randn(2, 300, 4, 64, generator=g, device="cuda") for _ in range(4)]
y = [t.bfloat16() for t in x]
w = torch.randn(2, 300, 200, generator=g, device="cuda")
z, ids, n = torch.randn(5, 32000, generator=g, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, device="cuda")
def run():
    r = []
    for q, k, v, d in (x, y):
        out, lse = training.attention_forward(q, k, v)
        r += [out, lse, *training.attention_backward(d, q, k, v, out, lse)]
    return r + [training.orthogonalise(w), training.orthogonalise(w[:, :40]), *training.policy_loss(z, ids, n, n)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
del got, graph
print("done")
"""
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    p = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "done" in p.stdout, p.stdout + p.stderr


# ---- scores that are no numbers -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 33])
@pytest.mark.parametrize("n", [90, 300])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_scores_that_are_no_numbers_stay_in_their_rows(dtype, dim, n, what):
    """A query's reach its own row, a key's the rows that see it (an infinite score leaves a row no finite sum either)."""
    g = gen(17)
    q, k, v = (rand(g, 2, n, 2, dim, dtype=dtype) for _ in range(3))
    out, lse = training.attention_forward(q, k, v)
    hit = torch.zeros(2, n, 2, dtype=torch.bool, device="cuda")
    q[0, 40, 1], k[1, n - 20, 0, 0] = what, what
    hit[0, 40, 1], hit[1, n - 20:, 0] = True, True
    if what == math.inf:
        q[1, n - 20:, 0, 0] = q[1, n - 20:, 0, 0].abs() + 1  # a score of +infinity in the rows that see it
        out, lse = training.attention_forward(q, torch.where(torch.isfinite(k), k, torch.ones_like(k)), v)
    got, sums = training.attention_forward(q, k, v)
    assert bool(got[hit].isnan().all()) and bool(sums.transpose(1, 2)[hit].isnan().all())
    assert torch.equal(got[~hit], out[~hit]) and torch.equal(sums.transpose(1, 2)[~hit], lse.transpose(1, 2)[~hit])
