"""The training operators against their definitions in 64 bits, through litnicelm_b200.training."""
import math

import pytest
import torch

from litnicelm_b200 import training
from train_ops_util import attention_reference, check, loss_reference, newton_schulz

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def fused(g, streams, n, m, heads, groups, dim, dtype):
    """q from one buffer, k and v from another, as slices of projected rows."""
    q = rand(g, streams, n, heads, dim, dtype=dtype)
    kv = rand(g, streams, m, 2 * groups, dim, dtype=dtype)
    return q, kv[:, :, :groups], kv[:, :, groups:]


def attention_case(dtype, streams, n, m, heads, groups, dim, seed=0, lengths=None, **opts):
    g = gen(seed)
    q, k, v = fused(g, streams, n, m, heads, groups, dim, dtype)
    dout = rand(g, streams, n, heads, dim, dtype=dtype)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = training.attention_forward(q, k, v, lengths=lens, **opts)
    dq, dk, dv = training.attention_backward(dout, q, k, v, out, lse, lengths=lens, **opts)
    ref = attention_reference(q, k, v, dout, lengths=lens, rounded=dtype == BF16, **opts)
    for name, got in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
        check(name, got, ref[name])


SIZES = [(1, 1, 1, 1, 1, 8), (2, 5, 5, 2, 1, 16), (1, 64, 64, 2, 2, 32), (2, 63, 63, 3, 3, 64), (1, 65, 65, 4, 2, 64),
         (2, 128, 128, 2, 2, 64), (1, 129, 129, 4, 1, 128), (1, 250, 250, 8, 8, 64), (3, 191, 191, 2, 1, 40),
         (1, 257, 257, 2, 2, 96), (1, 700, 700, 2, 1, 64), (1, 515, 515, 2, 2, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_attention_causal(dtype, size):
    attention_case(dtype, *size)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m,opts", [
    (70, 300, dict(causal=False)), (300, 70, dict(causal=False)), (1, 500, dict(first=499)), (130, 400, dict(first=270)),
    (200, 100, dict(first=0)), (100, 300, dict(first=10)), (300, 300, dict(window=1)), (300, 300, dict(window=37)),
    (400, 400, dict(window=128)), (300, 300, dict(window=100, causal=False)), (260, 130, dict(window=5)),
    (1, 1, dict(window=1)), (3, 200, dict(first=400, window=250)), (150, 90, dict(first=1000, window=3)),
    (64, 64, dict(scale=0.0)), (90, 90, dict(scale=-0.2)), (140, 140, dict(scale=1.7))], ids=str)
def test_attention_spans(dtype, n, m, opts):
    attention_case(dtype, 2, n, m, 4, 2, 64, **opts)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 24, 33, 48, 72, 80, 100, 120, 127, 128])
def test_attention_head_dimensions(dtype, dim):
    attention_case(dtype, 2, 77, 77, 2, 1, dim)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("opts", [dict(), dict(causal=False), dict(window=40), dict(window=40, causal=False)], ids=str)
def test_attention_lengths(dtype, dim, opts):
    attention_case(dtype, 7, 200, 200, 2, 2, dim, lengths=[200, 0, 1, 64, 65, 128, 199], **opts)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m,dim,lengths,opts", [
    (2100, 2100, 64, [2100, 1, 0, 2049], dict()), (2049, 2300, 40, [2300, 129, 1700, 64], dict(causal=False)),
    (2305, 2177, 64, [2177, 128, 2048, 0], dict(window=2060, causal=False)), (2176, 2400, 8, None, dict(first=200, window=2100)),
    (1100, 1200, 128, [1200, 65, 0, 1025], dict(first=100))], ids=str)
def test_attention_long(dtype, n, m, dim, lengths, opts):
    attention_case(dtype, 4, n, m, 2, 1, dim, lengths=lengths, **opts)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m,opts", [
    (300, 300, dict(scale=-0.2)), (300, 300, dict(scale=0.0)), (129, 700, dict(causal=False, scale=1.5)), (300, 500, dict(window=200)),
    (257, 600, dict(first=340, window=129)), (400, 300, dict(first=5, window=150)), (700, 130, dict(window=129)),
    (256, 129, dict(causal=False)), (390, 900, dict(first=510)), (700, 2, dict())], ids=str)
def test_attention_two_row_tiles(dtype, n, m, opts):
    attention_case(dtype, 3, n, m, 4, 2, 56, lengths=[m, 1, max(1, m - 130)], **opts)


@pytest.mark.parametrize("streams,n,opts", [(40, 200, dict()), (24, 300, dict(window=50)), (6, 1500, dict(causal=False))], ids=str)
def test_attention_calls_at_once(streams, n, opts):
    """Passes on two streams at the same time, and a captured one replayed beside an eager one, have the results of each by itself."""
    g = gen(31)
    lens = torch.randint(0, n + 1, (streams,), generator=g, device="cuda", dtype=torch.int32)
    sets = [(*fused(g, streams, n, n, 4, 2, 64, BF16), rand(g, streams, n, 4, 64, dtype=BF16)) for _ in range(2)]

    def both(q, k, v, dout):
        out, lse = training.attention_forward(q, k, v, lengths=lens, **opts)
        return (out, lse, *training.attention_backward(dout, q, k, v, out, lse, lengths=lens, **opts))

    alone = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams_at_once = [torch.cuda.Stream() for _ in sets]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both(*sets[0])
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams_at_once):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append([both(*s) for _ in range(3)][-1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(alone + alone[:1], got + [captured]):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [48, 128])
@pytest.mark.parametrize("opts", [dict(), dict(causal=False), dict(window=60), dict(first=300)], ids=str)
def test_attention_many_tiles(dtype, dim, opts):
    """More tiles than a GPU has multiprocessors, many of them without work, in runs and between others."""
    lengths = [300, 0, 0, 0, 0, 129, 1, 0, 300, 128, 0, 64, 0, 0, 257, 300, 2, 0, 300, 0, 0, 0, 0, 0]
    attention_case(dtype, 24, 300, 300, 8, 4, dim, lengths=lengths, **opts)


@pytest.mark.parametrize("dim", [40, 64, 128])
def test_attention_rows_of_one_key(dim):
    """Their weights are 1 whatever the scores: gradients of q and k are what 32-bit sums leave of nothing, however out was rounded.

    ds = scale p (dp - delta), delta = p dp: sums of dim products in two orders, each off by 2 dim u of the sum of magnitudes,
    and weights that are off by the score's error, twice (in lse too), and a few u."""
    g = gen(7)
    q, k, v = fused(g, 2, 300, 300, 4, 2, dim, BF16)
    dout = rand(g, 2, 300, 4, dim, dtype=BF16)
    out, lse = training.attention_forward(q, k, v, window=1)
    dq, dk, _ = training.attention_backward(dout, q, k, v, out, lse, window=1)
    u, scale = 2.0 ** -24, dim ** -0.5
    Q, D, K, V = q.double(), dout.double(), k.double().repeat_interleave(2, 2), v.double().repeat_interleave(2, 2)
    score, dp = (Q.abs() * K.abs()).sum(-1) * scale, (D.abs() * V.abs()).sum(-1)
    ds = scale * dp * (2 * 2 * dim * u + 2 * (2 * (dim + 4) * u * score + 16 * u + 8 * u * lse.transpose(1, 2).double().abs()))
    up = 1 + 2.0 ** -7  # to bfloat16, of ds and of the result
    assert bool((dq.double().abs() <= ds[..., None] * K.abs() * up + 1e-37).all())
    assert bool((dk.double().abs() <= (ds[..., None] * Q.abs()).view(2, 300, 2, 2, dim).sum(3) * up + 1e-37).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_no_work(dtype):
    attention_case(dtype, 40, 130, 130, 8, 8, 64, lengths=[0] * 40)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_hidden_lowest_values(dtype, dim):
    """The type's lowest value in keys and values that the span hides from every row."""
    g = gen(5)
    q, dout = (rand(g, 2, 60, 2, dim, dtype=dtype) for _ in range(2))
    k, v = (rand(g, 2, 100, 2, dim, dtype=dtype) for _ in range(2))
    results = []
    for x in (0.0, torch.finfo(dtype).min):
        k[:, 60:] = x
        v[:, 60:] = x
        out, lse = training.attention_forward(q, k, v)
        results.append((out, lse, *training.attention_backward(dout, q, k, v, out, lse)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf, "lowest"])
def test_attention_padding_is_not_used(dtype, what):
    """What lies behind a stream's length, in keys and values, reaches nothing."""
    g = gen(3)
    lengths = torch.tensor([100, 33, 0, 128], dtype=torch.int32, device="cuda")
    q, k, v = (rand(g, 4, 160, 2, 64, dtype=dtype) for _ in range(3))
    dout = rand(g, 4, 160, 2, 64, dtype=dtype)
    fill = torch.finfo(dtype).min if what == "lowest" else what
    results = []
    for x in (0.0, fill):
        for b, n in enumerate(lengths.tolist()):
            k[b, n:] = x
            v[b, n:] = x
        out, lse = training.attention_forward(q, k, v, lengths=lengths)
        results.append((out, lse, *training.attention_backward(dout, q, k, v, out, lse, lengths=lengths)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    out, lse, dq, dk, dv = results[0]
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all()) and bool((dq[2] == 0).all())
    for b, n in enumerate(lengths.tolist()):
        assert bool((dk[b, n:] == 0).all()) and bool((dv[b, n:] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_strides(dtype):
    """Heads before rows, columns apart, a shared (broadcast) key head, gradients into slices of one buffer."""
    g = gen(5)
    streams, n, heads, dim = 2, 150, 4, 64
    base = [rand(g, streams, heads, n, dim, dtype=dtype) for _ in range(4)]
    q, k, v, dout = (x.transpose(1, 2) for x in base)
    apart = [torch.empty(streams, n, heads, 2 * dim, dtype=dtype, device="cuda") for _ in range(3)]
    forms = [(q, k, v, dout)]
    for x, y in zip(apart, (q, k, v)):
        x[..., ::2] = y
    forms.append((*(x[..., ::2] for x in apart), dout.contiguous()))
    odd = torch.empty(streams * n * heads * dim + 1, dtype=dtype, device="cuda")[1:].view(streams, n, heads, dim)
    odd.copy_(q)  # on an odd element boundary
    forms.append((odd, k.contiguous(), v, dout))
    wide = torch.empty(streams, n, heads, dim + 3, dtype=dtype, device="cuda")[..., :dim]
    wide.copy_(k)  # rows that are no multiple of 16 bytes apart
    forms.append((q, wide, v, dout))
    ref = attention_reference(q, k, v, dout, rounded=dtype == BF16)
    for q1, k1, v1, d1 in forms:
        buffer = torch.full((streams, n, 3 * heads + 1, dim), 7.0, dtype=dtype, device="cuda")
        out, lse = training.attention_forward(q1, k1, v1)
        got = training.attention_backward(d1, q1, k1, v1, out, lse, dq=buffer[:, :, :heads], dk=buffer[:, :, heads:2 * heads],
                                          dv=buffer[:, :, 2 * heads:3 * heads])
        for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got)):
            check(name, x, ref[name])
        assert bool((buffer[:, :, 3 * heads:] == 7).all())
    k2, v2 = k[:, :, :1].expand(-1, -1, 2, -1), v[:, :, :1].expand(-1, -1, 2, -1)
    out, lse = training.attention_forward(q, k2, v2)
    got = training.attention_backward(dout, q, k2, v2, out, lse)
    ref = attention_reference(q, k2, v2, dout, rounded=dtype == BF16)
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got)):
        check(name, x, ref[name])


def test_attention_gradient_by_differences():
    """Against differences of the forward definition in 64 bits, not against the formula of the gradient."""
    g = gen(11)
    q, k, v = fused(g, 1, 20, 20, 2, 1, 8, F32)
    dout = rand(g, 1, 20, 2, 8)
    out, lse = training.attention_forward(q, k, v, window=9)
    grads = training.attention_backward(dout, q, k, v, out, lse, window=9)

    def value(*x):
        return float((attention_reference(*x, window=9)["out"][0] * dout.double()).sum())

    inputs = [x.double() for x in (q, k, v)]
    for which, (x, d) in enumerate(zip(inputs, grads)):
        turn = rand(g, *x.shape).double()
        h = 1e-5
        moved = [[y + s * h * turn if i == which else y for i, y in enumerate(inputs)] for s in (1, -1)]
        slope = (value(*moved[0]) - value(*moved[1])) / (2 * h)
        # the central difference is off by h^2 times a third derivative of order 1e2, the gradient by 1e-5 of its terms
        assert abs(slope - float((d.double() * turn).sum())) <= 1e-5 * (1 + float((d.double() * turn).abs().sum()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_large_scores(dtype):
    """Scores of several hundred: no overflow, rows whose weight sits on one key."""
    g = gen(13)
    q, k, v = fused(g, 1, 180, 180, 2, 2, 64, dtype)
    q, dout = (q * 30).to(dtype), rand(g, 1, 180, 2, 64, dtype=dtype)
    out, lse = training.attention_forward(q, k, v)
    got = training.attention_backward(dout, q, k, v, out, lse)
    ref = attention_reference(q, k, v, dout, rounded=dtype == BF16)
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *got)):
        check(name, x, ref[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_same_bits_every_time(dtype):
    g = gen(17)
    q, k, v = fused(g, 2, 600, 600, 8, 2, 64, dtype)
    dout = rand(g, 2, 600, 8, 64, dtype=dtype)
    out, lse = training.attention_forward(q, k, v)
    first = (out, lse, *training.attention_backward(dout, q, k, v, out, lse))
    for _ in range(3):
        o, s = training.attention_forward(q, k, v)
        for a, b in zip(first, (o, s, *training.attention_backward(dout, q, k, v, o, s))):
            assert torch.equal(a, b)


def test_attention_far_offsets():
    """Element offsets beyond 32 bits, in a buffer of which only the last rows are read."""
    rows = (1 << 31) // (8 * 64) + 300
    buffer = torch.empty(1, rows, 8, 64, dtype=BF16, device="cuda")
    g = gen(19)
    x = rand(g, 1, 140, 8, 64, dtype=BF16)
    buffer[:, -140:] = x
    q, k, v = buffer[:, -140:, :4], buffer[:, -140:, 4:6], buffer[:, -140:, 6:]
    far = torch.as_strided(buffer, (2, 140, 4, 64), ((rows - 140) * 512, 512, 64, 1))
    far[0] = x[0, :, :4]
    k2, v2 = (y.expand(2, -1, -1, -1) for y in (k, v))
    out, lse = training.attention_forward(far, k2, v2)
    ref = attention_reference(far, k2, v2, rounded=True)
    check("out", out, ref["out"])
    check("lse", lse, ref["lse"])
    del buffer, far, q, k, v


# ---- policy loss ---------------------------------------------------------------------------------------------------------------


def loss_case(dtype, rows, vocab, seed=0, kl=0.1, masked=True, temp=1.0, ld=None, spread=2.0, in_place=False, low=0.2, high=0.28):
    g = gen(seed)
    ld = ld or vocab
    logits = (rand(g, rows, ld) * spread).to(dtype)[:, :vocab]
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    now = torch.log_softmax(logits.double() / temp, 1).gather(1, targets.long()[:, None])[:, 0]
    old, refp = ((now + s * rand(g, rows).double()).float() for s in (0.3, 0.4))
    adv = rand(g, rows)
    weight = (torch.rand(rows, generator=g, device="cuda") < 0.7).float() * 1.5 if masked else None
    ref = loss_reference(logits, targets, old, adv, ref=refp if kl else None, weight=weight, temp=temp, low=low, high=high, kl=kl)
    loss, logp, d = training.policy_loss(logits, targets, old, adv, ref_logp=refp if kl else None, weight=weight, temp=temp,
                                         clip_low=low, clip_high=high, kl_weight=kl, dlogits=logits if in_place else None)
    assert not in_place or d.data_ptr() == logits.data_ptr()
    check("loss", loss, ref["loss"])
    check("logp", logp, ref["logp"])
    keep = ~ref["near"]
    check("dlogits", d[keep], tuple(x[keep] for x in ref["dlogits"]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 8), (3, 7), (64, 8), (250, 96), (33, 1000), (17, 1023), (5, 32000), (160, 32000),
                                        (2, 32771), (3, 57000), (2, 130001), (1, 300008), (2000, 96), (1, 2), (149, 4097)])
def test_policy_loss(dtype, rows, vocab):
    loss_case(dtype, rows, vocab)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("more", [dict(kl=0.0), dict(masked=False), dict(temp=0.7), dict(temp=3.0), dict(ld=1003), dict(ld=1008),
                                  dict(spread=30.0), dict(in_place=True), dict(in_place=True, ld=1003), dict(low=0.0, high=0.0),
                                  dict(low=1.0, high=1e30), dict(kl=-0.3)], ids=str)
def test_policy_loss_forms(dtype, more):
    loss_case(dtype, 70, 1000, **more)
    if "ld" not in more:
        loss_case(dtype, 4, 32000, **more)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [96, 1001, 32000, 70000])
def test_policy_loss_masked_rows_are_not_read(dtype, vocab):
    g = gen(2)
    logits = rand(g, 6, vocab, dtype=dtype)
    targets = torch.randint(0, vocab, (6,), generator=g, device="cuda", dtype=torch.int32)
    old, adv, ref = (rand(g, 6) for _ in range(3))
    weight = torch.tensor([1.0, 0, 2, 0, 0, 1], device="cuda")
    good = training.policy_loss(logits, targets, old, adv, ref_logp=ref, weight=weight, kl_weight=0.1)
    off = weight == 0
    logits[off] = math.nan
    targets[off] = -100
    old[off], adv[off], ref[off] = math.nan, math.inf, math.nan
    again = training.policy_loss(logits, targets, old, adv, ref_logp=ref, weight=weight, kl_weight=0.1)
    for a, b in zip(good, again):
        assert torch.equal(a, b)
    assert bool((again[1][off] == 0).all()) and bool((again[2][off] == 0).all())
    nothing = training.policy_loss(logits, targets, old, adv, weight=torch.zeros(6, device="cuda"))
    assert all(bool((x == 0).all()) for x in nothing)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [97, 32000])
def test_policy_loss_masked_places_and_bad_targets(dtype, vocab):
    """Logits of minus infinity or the type's lowest value have probability 0; a bad target is NaN in its row and the loss only."""
    g = gen(4)
    logits = rand(g, 4, vocab, dtype=dtype)
    logits[:, 1::3] = -math.inf
    logits[:, 2::3] = torch.finfo(dtype).min
    targets = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device="cuda")
    old, adv = -4 + 0.1 * rand(g, 4), rand(g, 4)
    ref = loss_reference(logits, targets, old, adv)
    loss, logp, d = training.policy_loss(logits, targets, old, adv)
    check("loss", loss, ref["loss"])
    check("logp", logp, ref["logp"])
    keep = ~ref["near"]
    check("dlogits", d[keep], tuple(x[keep] for x in ref["dlogits"]))
    assert bool((d[:, 1::3] == 0).all())
    for wrong in (-1, vocab, 2 ** 31 - 1):
        targets[2] = wrong
        loss, logp2, d2 = training.policy_loss(logits, targets, old, adv)
        assert math.isnan(float(loss)) and math.isnan(float(logp2[2])) and bool(d2[2].isnan().all())
        others = torch.tensor([0, 1, 3], device="cuda")
        assert torch.equal(logp2[others], logp[others]) and torch.equal(d2[others], d[others])
    logits[1] = -math.inf  # a row that is masked altogether is not a distribution
    targets[2] = 6
    loss, logp2, d2 = training.policy_loss(logits, targets, old, adv)
    assert math.isnan(float(loss)) and math.isnan(float(logp2[1])) and bool(d2[1].isnan().all()) and torch.equal(d2[0], d[0])


def test_policy_loss_forward_alone_and_same_bits():
    g = gen(6)
    logits = rand(g, 300, 5000)
    targets = torch.randint(0, 5000, (300,), generator=g, device="cuda", dtype=torch.int32)
    old, adv = -9 + rand(g, 300), rand(g, 300)
    a = training.policy_loss(logits, targets, old, adv, gradient=False)
    b = training.policy_loss(logits, targets, old, adv)
    c = training.policy_loss(logits, targets, old, adv)
    assert a[2] is None and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(x, y) for x, y in zip(b, c))


def test_policy_loss_gradient_by_differences():
    g = gen(8)
    logits = rand(g, 12, 40)
    targets = torch.randint(0, 40, (12,), generator=g, device="cuda", dtype=torch.int32)
    now = torch.log_softmax(logits, 1).gather(1, targets.long()[:, None])[:, 0]
    old, ref, adv = now + 0.05 * rand(g, 12), now + 0.3 * rand(g, 12), rand(g, 12)
    d = training.policy_loss(logits, targets, old, adv, ref_logp=ref, kl_weight=0.3, temp=1.3, clip_low=0.9, clip_high=9.0)[2]
    turn = rand(g, 12, 40).double()

    def value(s):
        return float(loss_reference(logits.double() + s * turn, targets, old, adv, ref=ref, kl=0.3, temp=1.3, low=0.9,
                                    high=9.0)["loss"][0])

    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    assert abs(slope - float((d.double() * turn).sum())) <= 1e-5 * (1 + float((d.double() * turn).abs().sum()))


# ---- orthogonalised momentum -----------------------------------------------------------------------------------------------------


def near_as_plain(got, u, steps=5):
    """No further from 64 bits than three times the same iteration with torch's 32-bit products, which round as often."""
    ref = newton_schulz(u.double(), steps)
    plain = newton_schulz(u, steps).double()
    norm = torch.linalg.matrix_norm(ref).clamp_min(1e-300)
    here = torch.linalg.matrix_norm(got.double() - ref) / norm
    there = torch.linalg.matrix_norm(plain - ref) / norm
    assert bool((here <= 3 * there + 8 * 2.0 ** -24).all()), (here.tolist(), there.tolist())


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (5, 3), (16, 16), (64, 256), (256, 64), (2, 3, 33, 65), (127, 129), (128, 128),
                                   (3, 200, 100), (613, 320), (4, 65, 400), (512, 2048), (1100, 700)], ids=str)
def test_orthogonalise(shape):
    g = gen(sum(shape))
    u = rand(g, *shape) * 0.01
    near_as_plain(training.orthogonalise(u), u)


@pytest.mark.parametrize("steps", [0, 1, 2, 7])
@pytest.mark.parametrize("shape", [(40, 70), (300, 200)])
def test_orthogonalise_steps(steps, shape):
    u = rand(gen(steps), *shape)
    near_as_plain(training.orthogonalise(u, steps=steps), u, steps)


def test_orthogonalise_scales_and_zeros():
    """Any size of input, matrices of one call that differ in it, low rank, zero matrices, the place of the input itself."""
    g = gen(9)
    for shape in ((96, 150), (300, 260)):
        u = rand(g, 5, *shape)
        u[0] *= 1e-18
        u[1] *= 1e18
        u[2] = 0
        u[3] = rand(g, shape[0], 1) @ rand(g, 1, shape[1])
        got = training.orthogonalise(u)
        assert bool((got[2] == 0).all())
        near_as_plain(got[[1, 3, 4]], u[[1, 3, 4]])
        near_as_plain(got[:1], u[:1])
        v = u.clone()
        assert training.orthogonalise(v, out=v) is v and torch.equal(v, got)


@pytest.mark.parametrize("shape", [(2, 40, 70), (2, 96, 152), (300, 260), (2, 130, 99)], ids=str)
@pytest.mark.parametrize("power", [-20, 60, 120])
def test_orthogonalise_powers_of_two(shape, power):
    """A power of two changes nothing but what 1e-7 beside the norm is worth (2^-20 of a norm above 50: 2e-3 of a factor, which the
    iteration forgets no faster than it magnifies it, a factor of 3.4445 a step) and roundings of x, 2^-23 of an element."""
    u = rand(gen(5), *shape)
    one, other = training.orthogonalise(u).double(), training.orthogonalise(u * 2.0 ** power).double()
    norm = torch.linalg.matrix_norm(u.double()).min()
    part = 1e-7 / float(norm) * max(1.0, 2.0 ** -power) + 4 * 2.0 ** -23
    off = torch.linalg.matrix_norm(one - other) / torch.linalg.matrix_norm(one)
    assert bool((off <= 3.4445 ** 5 * part).all()) and bool(torch.isfinite(other).all())


def test_orthogonalise_strides():
    g = gen(10)
    big = rand(g, 3, 90, 2, 130)
    x = big[:, ::2, 1, 1::2]
    out = torch.zeros(3, 65, 45, device="cuda").mT
    got = training.orthogonalise(x, out=out)
    assert got is out and torch.equal(out, training.orthogonalise(x.contiguous()))
    near_as_plain(out, x.contiguous())
    assert torch.equal(training.orthogonalise(x[0]), out[0]) or float((training.orthogonalise(x[0]) - out[0]).abs().max()) < 1e-5


@pytest.mark.parametrize("shape", [(64, 256), (2, 300, 130), (3, 31, 33)], ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(shape, nesterov):
    g = gen(21)
    params, grads, momentum = (rand(g, *shape) for _ in range(3))
    params *= 0.02
    p, m = params.clone(), momentum.clone()
    training.muon_step(p, grads, m, 0.03, mu=0.9, weight_decay=0.1, nesterov=nesterov)
    m64 = 0.9 * momentum.double() + grads.double()
    # mu is 0.9 rounded to 32 bits, the sum is rounded once
    assert bool(((m.double() - m64).abs() <= 2 * 2.0 ** -24 * ((0.9 * momentum).abs() + m.abs()).double() + 1e-37).all())
    u = (grads + 0.9 * m if nesterov else m).float()
    x = newton_schulz(u.double())
    rate = 0.03 * math.sqrt(max(1, shape[-2] / shape[-1]))
    want = params.double() * (1 - 0.03 * 0.1) - rate * x
    off = torch.linalg.matrix_norm(newton_schulz(u).double() - x) * rate
    assert bool((torch.linalg.matrix_norm(p.double() - want) <= 3 * off + 8 * 2.0 ** -24 * torch.linalg.matrix_norm(want)).all())


# ---- streams, graphs, and a step of all of them --------------------------------------------------------------------------------------


def test_calls_on_another_stream_and_in_graphs():
    """Captured twice, replayed on new inputs beside each other's workspaces and an eager call."""
    g = gen(30)
    n, vocab = 200, 1000
    x = [rand(g, 1, n, 4, 64, dtype=BF16) for _ in range(4)]
    logits, adv, old = rand(g, n, vocab), rand(g, n), -7 + rand(g, n)
    targets = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    w = rand(g, 2, 70, 150)

    def work():
        out, lse = training.attention_forward(*x[:3])
        return (out, lse, *training.attention_backward(x[3], *x[:3], out, lse),
                *training.policy_loss(logits, targets, old, adv, weight=(adv > -1).float()), training.orthogonalise(w))

    plain = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(plain, other))
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(work())
        graphs.append(graph)
    for y in (*x, logits, w):
        y.mul_(0.5)
    plain = work()
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    eager = work()
    torch.cuda.synchronize()
    for r in (*results, eager):
        assert all(torch.equal(a, b) for a, b in zip(plain, r))
    # graphs let go of their memory before the process ends
    del results, graphs


def test_between_calls_of_the_table():
    """On a table instance's own stream: behind the calls it has recorded, before those that follow."""
    from litnicelm_b200.plugin import Backend, DevTensor
    g = gen(31)
    with Backend() as be:
        a, b, c = (rand(g, 40, 60) for _ in range(3))
        torch.cuda.synchronize()

        def view(t):
            return DevTensor(t.data_ptr(), tuple(t.shape), tuple(4 * s for s in t.stride()))

        be.call("add", view(a), view(b), view(c))
        with torch.cuda.stream(torch.cuda.ExternalStream(be.stream())):
            d = training.orthogonalise(c)
        be.call("add", view(d), view(b), view(c))
        be.stream()
        torch.cuda.synchronize()
        near_as_plain(d, a + b)
        assert torch.equal(c, d + b)


def test_training_step_of_a_layer():
    """Attention, loss and optimiser together as a step uses them, against the same step in 64 bits by torch's own gradients."""
    g = gen(40)
    streams, n, width, heads, vocab = 3, 50, 64, 4, 96
    x = rand(g, streams, n, width)
    wqkv, head = rand(g, width, 3 * width) / 8, rand(g, width, vocab) / 8
    lengths = torch.tensor([50, 31, 1], dtype=torch.int32, device="cuda")
    weight = (torch.arange(n, device="cuda")[None] < lengths[:, None]).float().flatten()
    targets = torch.randint(0, vocab, (streams * n,), generator=g, device="cuda", dtype=torch.int32)
    adv, old, ref = rand(g, streams * n), -4.5 + 0.2 * rand(g, streams * n), -4.5 + 0.2 * rand(g, streams * n)
    mom = [torch.zeros_like(wqkv), torch.zeros_like(head)]

    def split(rows):
        return [r.reshape(streams, n, heads, width // heads) for r in rows.split(width, -1)]

    reference = [wqkv.double().requires_grad_(), head.double().requires_grad_()]
    seen = (torch.arange(n, device="cuda")[None, :, None] >= torch.arange(n, device="cuda")[None, None, :]) & \
        (torch.arange(n, device="cuda")[None, None, :] < lengths[:, None, None])
    q, k, v = (t.transpose(1, 2) for t in split(x.double() @ reference[0]))
    p = torch.softmax((q @ k.mT / math.sqrt(width // heads)).masked_fill(~seen[:, None], -math.inf), -1)
    z = (p @ v).transpose(1, 2).reshape(streams * n, width) @ reference[1]
    logp = torch.log_softmax(z, 1).gather(1, targets.long()[:, None])[:, 0]
    r, d = torch.exp(logp - old), ref - logp
    rows = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (torch.exp(d) - d - 1)
    loss = (rows * weight).sum() / weight.sum()
    loss.backward()

    qkv = x @ wqkv
    q, k, v = split(qkv)
    out, lse = training.attention_forward(q, k, v, lengths=lengths)
    flat = out.reshape(streams * n, width)
    got, _, dlogits = training.policy_loss(flat @ head, targets, old, adv, ref_logp=ref, weight=weight, kl_weight=0.1)
    dout = (dlogits @ head.t()).reshape(out.shape)
    dqkv = torch.empty_like(qkv)
    dq, dk, dv = split(dqkv)
    training.attention_backward(dout, q, k, v, out, lse, lengths=lengths, dq=dq, dk=dk, dv=dv)
    grads = [x.reshape(-1, width).t() @ dqkv.reshape(-1, 3 * width), flat.t() @ dlogits]
    assert abs(float(got) - float(loss)) <= 1e-5 * (1 + float((rows.abs() * weight).sum() / weight.sum()))
    for a, b in zip(grads, reference):
        # chains of four 32-bit products of up to 192 terms: a few times 192 u of the largest entries
        assert float((a - b.grad).abs().max()) <= 1e-4 * float(b.grad.abs().max())
    before = [wqkv.clone(), head.clone()]
    for w, d, m, b in zip((wqkv, head), grads, mom, before):
        training.muon_step(w, d, m, 0.02, nesterov=False)
        assert torch.equal(m, d)
        step = (b - w) / (0.02 * math.sqrt(max(1, w.shape[0] / w.shape[1])))
        values = torch.linalg.svdvals(step.double())
        assert float(values.max()) < 1.3 and float(values.median()) > 0.6
