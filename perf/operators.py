"""Operators of a training step, as cases that can be timed and checked: attention with its backward pass, a clipped policy
loss with its gradient, and the update of weight matrices by orthogonalised momentum.

Families of cases, each through the public entry points of ``litnicelm_b200.training``:

* ``attention``  ``attention_forward`` and, where ``backward`` is set, ``attention_backward`` on its results. Queries, keys and
                 values are slices of one buffer of projected rows, as a layer's projection leaves them. Key heads may be shared
                 by query heads, rows may see a window of the last keys only, and a padded batch brings its lengths.
* ``loss``       ``policy_loss``: loss, log probabilities and the gradient of the logits.
* ``muon``       ``muon_step`` on matrices of one shape: momentum, orthogonalisation, weights.
* ``orthogonal`` ``orthogonalise`` alone.

Sizes are those of the repository's configurations (widths 64, 512 and 1024, heads of 32 and 64, vocabularies of 96 and 32000,
texts of 64 to 2048 tokens), sizes between them, and longer texts and wider heads of the same kind.

``own`` false: the plain form, from elementary torch operations in 32 bits. ``exact``: the definition in 64 bits.
"""
import math

import torch

own = False

BF16, F32 = "bfloat16", "float32"


def _attention(name, dtype, streams, n, heads, groups, dim, window=0, padded=False, backward=True):
    return dict(family="attention", name=name, dtype=dtype, streams=streams, n=n, heads=heads, groups=groups, dim=dim, window=window,
                padded=padded, backward=backward)


def _loss(name, dtype, rows, vocab, kl=0.05, masked=True):
    return dict(family="loss", name=name, dtype=dtype, rows=rows, vocab=vocab, kl=kl, masked=masked)


def _matrices(name, family, count, m, n):
    return dict(family=family, name=name, count=count, m=m, n=n)


def listed():
    return [
        # a step of the smallest model: launches and latency
        _attention("attention-tiny", F32, 4, 64, 2, 2, 32),
        # the character model's layers in its own 32 bits, texts of no round length
        _attention("attention-char", F32, 8, 250, 8, 8, 64),
        # the large transformer's layer, in the 16-bit type of the registered designs
        _attention("attention-large", BF16, 4, 2048, 16, 16, 64),
        # a padded batch scored without training on it: forward alone, odd length
        _attention("attention-scored", BF16, 8, 1535, 16, 16, 64, padded=True, backward=False),
        # a long text through heads of 128 that share keys and values
        _attention("attention-long", BF16, 1, 8192, 16, 4, 128),
        # characters: a small vocabulary, every row
        _loss("loss-char", F32, 2000, 96, masked=False),
        # a batch of sampled texts over the large vocabulary, prompts masked
        _loss("loss-large", F32, 4096, 32000),
        _loss("loss-large-bf16", BF16, 4093, 32000, kl=0.0),
        # one small matrix, as the smallest model's projections
        _matrices("muon-tiny", "muon", 2, 64, 256),
        # all first feed-forward matrices of the character model
        _matrices("muon-char", "muon", 6, 512, 2048),
        # a group of the large transformer's feed-forward matrices, tall ones
        _matrices("muon-large", "muon", 4, 4096, 1024),
        # a matrix of no round size, the orthogonal factor alone
        _matrices("orthogonal-odd", "orthogonal", 1, 613, 1601),
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["attention", "attention", "loss", "muon", "orthogonal"])
    if family == "attention":
        dtype = rng.choice([F32, BF16, BF16])
        n = _between(rng, 1, 2048 if dtype == F32 else 6000)
        groups = rng.choice([1, 2, 4, 8])
        heads = groups * rng.choice([1, 1, 2, 4])
        dim = rng.choice([32, 64, 64, 128] + ([24, 40] if dtype == F32 else [16, 96]))
        # the pairs of a pass stay below those of the largest listed case; 32 bits a sixteenth of it
        room = (8192 * 8192 * 16 // (16 if dtype == F32 else 2)) // (n * n * heads)
        streams = max(1, min(rng.randint(1, 16), room))
        window = rng.choice([0, 0, _between(rng, 1, 2 * n)])
        case = _attention("", dtype, streams, n, heads, groups, dim, window, rng.random() < 0.4, rng.random() < 0.7)
    elif family == "loss":
        vocab = _between(rng, 8, 32000)
        rows = _between(rng, 1, min(16384, 4000 * 32000 // vocab))
        case = _loss("", rng.choice([F32, BF16]), rows, vocab, rng.choice([0.0, 0.02, 0.1]), rng.random() < 0.6)
    else:
        m, n = _between(rng, 16, 2048), _between(rng, 16, 4096)
        count = max(1, min(rng.randint(1, 8), 4 * 1024 * 1024 * 4096 // (min(m, n) ** 2 * max(m, n))))
        case = _matrices("", family, count, m, n)
    del case["name"]
    return case


# ---- what a user's program has in hand --------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["family"] == "attention":
        dtype = getattr(torch, case["dtype"])
        streams, n, heads, groups, dim = (case[k] for k in ("streams", "n", "heads", "groups", "dim"))
        rows = normal(streams, n, heads + 2 * groups, dim).to(dtype)
        s["q"], s["k"], s["v"] = rows[:, :, :heads], rows[:, :, heads:heads + groups], rows[:, :, heads + groups:]
        s["lengths"] = None
        if case["padded"]:  # the longest text fills its row; one may be empty
            lengths = torch.randint(0, n + 1, (streams,), generator=g, device="cuda", dtype=torch.int32)
            lengths[0] = n
            s["lengths"] = lengths
        s["dout"] = normal(streams, n, heads, dim).to(dtype) if case["backward"] else None
    elif case["family"] == "loss":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (normal(rows, vocab) * 2).to(getattr(torch, case["dtype"]))
        s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        # the targets were sampled: they are likelier than the others
        s["logits"].scatter_add_(1, s["targets"].long()[:, None], (3 + 2 * normal(rows, 1)).to(s["logits"].dtype))
        now = torch.log_softmax(s["logits"].float(), 1).gather(1, s["targets"].long()[:, None])[:, 0]
        s["old"] = now + 0.2 * normal(rows)          # the policy that sampled is a few steps behind
        s["ref"] = now + 0.3 * normal(rows) if case["kl"] else None
        s["advantage"] = normal(rows) + 0.25
        s["weight"] = (uniform(rows) < 0.7).float() if case["masked"] else None
    else:
        count, m, n = case["count"], case["m"], case["n"]
        # gradients of a layer have a few strong directions above the noise
        def gradient():
            return 1e-3 * (normal(count, m, n) + 4 * normal(count, m, 4) @ normal(count, 4, n) / 2)
        s["grads"] = gradient()
        if case["family"] == "muon":
            s["momentum"] = 5 * gradient()
            s["params"] = 0.02 * normal(count, m, n)
    return s


# ---- the operators -----------------------------------------------------------------------------------------------------------


LR, MU, DECAY, STEPS = 0.02, 0.95, 0.01, 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _seen(s, n, device):
    """[streams or 1, n, n]: which keys a row sees."""
    i = torch.arange(n, device=device)
    seen = i[None, :] <= i[:, None]
    if s["window"]:
        seen = seen & (i[None, :] > i[:, None] - s["window"])
    seen = seen[None]
    if s["lengths"] is not None:
        seen = seen & (i[None, None, :] < s["lengths"][:, None, None])
    return seen


def _plain_attention(s):
    share = s["heads"] // s["groups"]
    q = s["q"].float().transpose(1, 2)
    k, v = (s[x].float().transpose(1, 2).repeat_interleave(share, 1) for x in ("k", "v"))
    scale = 1 / math.sqrt(s["dim"])
    seen = _seen(s, s["n"], q.device)[:, None]
    scores = (q @ k.transpose(2, 3) * scale).masked_fill_(~seen, -math.inf)
    top = scores.amax(3, keepdim=True).clamp_min_(-3e38)
    p = (scores - top).exp_()
    del scores
    total = p.sum(3, keepdim=True)
    lse = (top + total.log())[..., 0]
    p = p / total.where(total > 0, torch.ones_like(total))
    out = p @ v
    dtype = s["q"].dtype
    got = {"out": out.transpose(1, 2).to(dtype), "lse": lse}
    if s["backward"]:
        dout = s["dout"].float().transpose(1, 2)
        shared = (s["streams"], s["groups"], share, s["n"], s["dim"])
        got["dv"] = (p.transpose(2, 3) @ dout).reshape(shared).sum(2).transpose(1, 2).to(dtype)
        ds = dout @ v.transpose(2, 3)
        ds = ds.sub_((dout * out).sum(3, keepdim=True)).mul_(p).mul_(scale)
        got["dq"] = (ds @ k).transpose(1, 2).to(dtype)
        got["dk"] = (ds.transpose(2, 3) @ q).reshape(shared).sum(2).transpose(1, 2).to(dtype)
    return got


def _plain_loss(s):
    z = s["logits"].float()
    at = s["targets"].long()[:, None]
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    logp = (z.gather(1, at) - top - total.log())[:, 0]
    weight = torch.ones_like(logp) if s["weight"] is None else s["weight"]
    per = weight / weight.double().sum().clamp_min(1e-30).float()
    ratio = (logp - s["old"]).exp()
    a = s["advantage"]
    rows = -torch.minimum(ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a)
    free = torch.where(a >= 0, ratio <= 1 + CLIP_HIGH, ratio >= 1 - CLIP_LOW)
    dlogp = torch.where(free, -ratio * a, torch.zeros_like(a))
    if s["kl"]:
        more = s["ref"] - logp
        rows = rows + s["kl"] * (more.exp() - more - 1)
        dlogp = dlogp + s["kl"] * (1 - more.exp())
    dlogp = torch.where(weight != 0, dlogp * per, torch.zeros_like(per))
    loss = (torch.where(weight != 0, rows * per, torch.zeros_like(per))).double().sum().float()
    d = e.mul_(-dlogp[:, None] / total)
    d.scatter_add_(1, at, dlogp[:, None])
    return {"loss": loss, "logp": logp * (weight != 0), "dlogits": d.to(s["logits"].dtype)}


def _plain_orthogonal(u):
    a, b, c = COEFFICIENTS
    norm = u.double().square().sum((1, 2), keepdim=True).sqrt().float()
    x = u / (norm + 1e-7)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        y = x @ x.transpose(1, 2)
        x = a * x + (b * y + c * (y @ y)) @ x
    return x.transpose(1, 2) if tall else x


def _plain_muon(s):
    momentum = s["momentum"].mul_(MU).add_(s["grads"])
    x = _plain_orthogonal(s["grads"] + MU * momentum)
    s["params"].mul_(1 - LR * DECAY).sub_(x * (LR * math.sqrt(max(1.0, s["m"] / s["n"]))))
    return {"params": s["params"], "momentum": momentum}


def run(state):
    s = state
    if own:
        from litnicelm_b200 import training

        if s["family"] == "attention":
            opts = dict(window=s["window"], lengths=s["lengths"])
            out, lse = training.attention_forward(s["q"], s["k"], s["v"], **opts)
            got = {"out": out, "lse": lse}
            if s["backward"]:
                got["dq"], got["dk"], got["dv"] = training.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **opts)
            return got
        if s["family"] == "loss":
            loss, logp, dlogits = training.policy_loss(s["logits"], s["targets"], s["old"], s["advantage"], ref_logp=s["ref"],
                                                       weight=s["weight"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_weight=s["kl"])
            return {"loss": loss, "logp": logp, "dlogits": dlogits}
        if s["family"] == "muon":
            training.muon_step(s["params"], s["grads"], s["momentum"], LR, mu=MU, weight_decay=DECAY, steps=STEPS)
            return {"params": s["params"], "momentum": s["momentum"]}
        return training.orthogonalise(s["grads"], steps=STEPS)
    if s["family"] == "attention":
        return _plain_attention(s)
    if s["family"] == "loss":
        return _plain_loss(s)
    if s["family"] == "muon":
        return _plain_muon(s)
    return _plain_orthogonal(s["grads"])


def work(case):
    if case["family"] == "attention":
        streams, n, heads, groups, dim, window = (case[k] for k in ("streams", "n", "heads", "groups", "dim", "window"))
        size = 2 if case["dtype"] == BF16 else 4
        w = min(window, n) if window else n
        pairs = w * (w + 1) // 2 + (n - w) * w  # a padded batch: about half of its keys, which the seed decides
        pairs = pairs * streams * heads * (0.5 if case["padded"] else 1.0)
        rows = streams * n
        q, kv, lse = rows * heads * dim * size, 2 * rows * groups * dim * size, rows * heads * 4
        if not case["backward"]:
            return {"bytes": 2 * q + kv + lse, "flops": 4 * dim * pairs}
        # inputs, upstream gradient, results: the forward pass's own are read again behind it
        return {"bytes": 4 * q + 2 * kv + lse, "flops": 14 * dim * pairs}
    if case["family"] == "loss":
        size = 2 if case["dtype"] == BF16 else 4
        rows = case["rows"]
        return {"bytes": 2 * rows * case["vocab"] * size + rows * 4 * (4 + (case["kl"] != 0) + case["masked"]),
                "flops": 6 * rows * case["vocab"]}
    p, q, count = min(case["m"], case["n"]), max(case["m"], case["n"]), case["count"]
    # the two symmetric products of a step need half of their results
    flops = count * STEPS * (p * p * q + p * p * p + 2 * p * p * q)
    return {"bytes": count * p * q * 4 * (5 if case["family"] == "muon" else 2), "flops": flops}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------


def _exact_attention(s):
    """Head by head: weights from the log-sum-exp, gradients from the chain rule."""
    out = torch.zeros(s["streams"], s["n"], s["heads"], s["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((s["streams"], s["heads"], s["n"]), -math.inf, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(s["streams"], s["n"], s["groups"], s["dim"], dtype=torch.float64, device="cuda") for _ in range(2))
    place = torch.arange(s["n"], device="cuda")
    gap = place[:, None] - place[None, :]
    for b in range(s["streams"]):
        keys = s["n"] if s["lengths"] is None else int(s["lengths"][b])
        if keys == 0:
            continue
        hidden = gap[:, :keys] < 0
        if s["window"]:
            hidden = hidden | (gap[:, :keys] >= s["window"])
        for h in range(s["heads"]):
            at = h * s["groups"] // s["heads"]
            q, k, v = s["q"][b, :, h].double(), s["k"][b, :keys, at].double(), s["v"][b, :keys, at].double()
            z = torch.where(hidden, torch.full_like(q[:1, :1], -math.inf), torch.mm(q, k.t()) / math.sqrt(s["dim"]))
            norm = torch.logsumexp(z, 1)
            lse[b, h] = norm
            p = torch.where(hidden, torch.zeros_like(z), torch.exp(z - norm[:, None]))
            out[b, :, h] = torch.mm(p, v)
            if s["backward"]:
                up = s["dout"][b, :, h].double()
                dv[b, :keys, at] += torch.mm(p.t(), up)
                dp = torch.mm(up, v.t())
                dz = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(s["dim"])
                dq[b, :, h] = torch.mm(dz, k)
                dk[b, :keys, at] += torch.mm(dz.t(), q)
    got = {"out": out, "lse": lse}
    return {**got, "dq": dq, "dk": dk, "dv": dv} if s["backward"] else got


def _exact_loss(s):
    """The gradient by the derivative of the row's loss in its log probability, times that of the log softmax."""
    rows, vocab = s["logits"].shape
    places = torch.arange(rows, device="cuda")
    target = s["targets"].long()
    full = torch.log_softmax(s["logits"].double(), dim=-1)
    logp = full[places, target]
    weight = torch.ones(rows, dtype=torch.float64, device="cuda") if s["weight"] is None else s["weight"].double()
    share = weight / torch.clamp(weight.sum(), min=1e-30)
    x = logp.clone().requires_grad_(True)
    adv = s["advantage"].double()
    r = torch.exp(x - s["old"].double())
    clipped = torch.clamp(r, 1 - CLIP_LOW, 1 + CLIP_HIGH)
    value = -torch.where(r * adv <= clipped * adv, r * adv, clipped * adv)
    if s["kl"]:
        d = s["ref"].double() - x
        value = value + s["kl"] * (torch.expm1(d) - d)
    loss = (value * share).sum()
    (slope,) = torch.autograd.grad(loss, x)
    grad = -torch.exp_(full) * slope[:, None]
    grad[places, target] += slope
    return {"loss": loss.detach(), "logp": torch.where(weight != 0, logp, torch.zeros_like(logp)), "dlogits": grad}


def _exact_orthogonal(u):
    """The polynomial of each step in the eigenvectors of the smaller Gram matrix: it acts on the singular values alone."""
    a, b, c = COEFFICIENTS
    u = u / (torch.linalg.matrix_norm(u, keepdim=True) + 1e-7)
    wide = u.shape[-1] >= u.shape[-2]
    gram = torch.matmul(u, u.mT) if wide else torch.matmul(u.mT, u)
    values, vectors = torch.linalg.eigh(gram)
    sigma2 = values.clamp_min(0)
    factor = torch.ones_like(sigma2)
    for _ in range(STEPS):
        step = a + sigma2 * (b + c * sigma2)
        factor, sigma2 = factor * step, sigma2 * step * step
    turn = torch.matmul(vectors * factor[..., None, :], vectors.mT)
    return torch.matmul(turn, u) if wide else torch.matmul(u, turn)


def exact(case, seed):
    s = prepare(case, seed)
    if s["family"] == "attention":
        return _exact_attention(s)
    if s["family"] == "loss":
        return _exact_loss(s)
    g = s["grads"].double()
    if s["family"] == "orthogonal":
        return _exact_orthogonal(g)
    momentum = MU * s["momentum"].double() + g
    x = _exact_orthogonal(g + MU * momentum)
    params = s["params"].double() * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, s["m"] / s["n"])) * x
    return {"params": params, "momentum": momentum}
