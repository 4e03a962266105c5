"""64-bit references of the training operators, with bounds on what 32-bit (and bfloat16) arithmetic may be off element by element.

u = 2^-24 is half a step of a 32-bit float. A sum of k terms on the tensor cores may truncate at each addition: 2 k u of the
sum of magnitudes. Exponentials are good to 8 u beside the error of their argument."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seen_keys(n, m, causal, first, window, lengths, streams, device):
    i = torch.arange(n, device=device)[:, None] + first
    j = torch.arange(m, device=device)[None, :]
    seen = torch.ones(n, m, dtype=torch.bool, device=device)
    if causal:
        seen = seen & (j <= i)
    if window:
        seen = seen & (j > i - window)
    seen = seen[None].expand(streams, n, m)
    if lengths is not None:
        seen = seen & (j[None] < lengths[:, None, None])
    return seen[:, None]


def attention_reference(q, k, v, dout=None, *, scale=None, causal=True, first=0, window=0, lengths=None, rounded=False):
    """{name: (value, bound)} in 64 bits. rounded: weights and their gradients may be rounded to bfloat16 for their products."""
    dtype, (streams, n, heads, dim), (m, groups) = q.dtype, q.shape, k.shape[1:3]
    share = heads // groups
    scale = 1 / math.sqrt(dim) if scale is None else scale
    seen = seen_keys(n, m, causal, first, window, lengths, streams, q.device)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    keys = torch.arange(m, device=q.device)[None, :, None, None]
    live = keys < (m if lengths is None else lengths[:, None, None, None])
    k, v = (torch.where(live, x.double(), zero) for x in (k, v))

    def heads_first(x):
        return x.double().transpose(1, 2)

    def shared(x):
        return heads_first(x).repeat_interleave(share, 1)

    def joined(x):
        return x.reshape(streams, groups, share, m, dim).sum(2).transpose(1, 2)

    Q, K, V = heads_first(q), shared(k), shared(v)
    s = Q @ K.transpose(2, 3) * scale
    es = (dim + 4) * 2 * U * abs(scale) * (Q.abs() @ K.abs().transpose(2, 3)) + 4 * U * s.abs()
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, 3)
    some = seen.any(3)
    safe = torch.where(some, lse, torch.zeros_like(lse))
    p = torch.where(seen, torch.exp(s - safe[..., None]), torch.zeros_like(s))
    # the weights' relative error: argument, exponential, and the sum that divides them
    et = torch.where(seen, es, torch.zeros_like(es)) + 8 * U + 4 * U * safe.abs()[..., None]
    el = (p * et).sum(3) + (m + 8) * U
    ew = et + el[..., None]
    round_w = half_step(torch.bfloat16) if rounded else 0.0
    h = half_step(dtype)
    out = p @ V
    eo = (p * (ew + round_w + 2 * m * U)) @ V.abs()
    ref = {"out": (out.transpose(1, 2), (eo + h * (out.abs() + eo)).transpose(1, 2) + 1e-37),
           "lse": (lse, torch.where(some, el + 4 * U * (1 + safe.abs()), torch.zeros_like(el)))}
    if dout is None:
        return ref
    D = heads_first(dout)
    dp = D @ V.transpose(2, 3)
    delta = (D * out).sum(3)
    edelta = (D.abs() * (eo + (h + 2 * dim * U) * (out.abs() + eo))).sum(3)
    ds = p * (dp - delta[..., None]) * scale
    eds = abs(scale) * p * (ew * (dp - delta[..., None]).abs() + 2 * (dim + 2) * U * (D.abs() @ V.abs().transpose(2, 3)) +
                            edelta[..., None] + 2 * U * delta.abs()[..., None]) + (round_w + 4 * U) * ds.abs()
    rows = n * share
    dq = ds @ K
    edq = (eds + 2 * m * U * ds.abs()) @ K.abs()
    dk = joined(ds.transpose(2, 3) @ Q)
    edk = joined((eds + 2 * rows * U * ds.abs()).transpose(2, 3) @ Q.abs())
    dv = joined(p.transpose(2, 3) @ D)
    edv = joined((p * (ew + round_w + 2 * rows * U)).transpose(2, 3) @ D.abs())
    ref["dq"] = (dq.transpose(1, 2), (edq + h * (dq.abs() + edq)).transpose(1, 2) + 1e-37)
    ref["dk"] = (dk, edk + h * (dk.abs() + edk) + 1e-37)
    ref["dv"] = (dv, edv + h * (dv.abs() + edv) + 1e-37)
    return ref


def loss_reference(logits, targets, old, adv, *, ref=None, weight=None, temp=1.0, low=0.2, high=0.2, kl=0.0):
    """{name: (value, bound)}; rows of weight 0 are left out of everything."""
    rows, vocab = logits.shape
    dtype = logits.dtype
    w = torch.ones(rows, dtype=torch.float64, device=logits.device) if weight is None else weight.double()
    on = w != 0
    z = torch.where(on[:, None], logits.double(), torch.zeros((), dtype=torch.float64, device=logits.device)) / temp
    at = torch.where(on, targets.long(), torch.zeros_like(targets.long()))[:, None]
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, at)[:, 0]
    logp = zt - lse
    top = z.amax(1)
    p = torch.exp(z - lse[:, None])
    gap = torch.where(torch.isfinite(z), (z - top[:, None]).abs(), torch.zeros_like(z))
    ee = 6 * U * gap + 8 * U                                   # of an exponential
    es = (p * ee).sum(1) + (vocab / 128 + 40) * U              # of their sum
    elog = es + 4 * U * ((zt - top).abs() + (lse - top).abs() + 1)
    r = torch.exp(logp - old.double())
    er = elog + 2 * U * (logp - old.double()).abs() + 4 * U
    a = adv.double()
    clipped = r.clamp(1 - low, 1 + high)
    value = -torch.minimum(r * a, clipped * a)
    free = torch.where(a >= 0, r <= 1 + high, r >= 1 - low)
    g = torch.where(free, -r * a, torch.zeros_like(a))
    ev, eg = (er + 4 * U) * (r * a).abs() + 4 * U * a.abs(), (er + 4 * U) * (r * a).abs()
    if kl:
        d = ref.double() - logp
        e = torch.exp(d)
        ed = elog + 2 * U * d.abs()
        value = value + kl * (torch.expm1(d) - d)
        g = g + kl * -torch.expm1(d)
        ev = ev + abs(kl) * (ed * (e - 1).abs() + 6 * U * (e + 1 + d.abs()))
        eg = eg + abs(kl) * (ed * e + 6 * U * (e + 1))
    near = torch.minimum((r - 1 - high).abs(), (r - 1 + low).abs()) <= 2 * er * r  # either branch is right there
    total = w.sum()
    share = torch.where(on, w / (total if total != 0 else 1.0), torch.zeros_like(w))
    loss = (share * torch.where(on, value, torch.zeros_like(value))).sum()
    eloss = (share * (ev + 4 * U * value.abs())).nan_to_num().sum() + 2 * U * loss.abs()
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    slope = torch.where(on, share * g, torch.zeros_like(g))
    eslope = torch.where(on, share * eg + 6 * U * slope.abs(), torch.zeros_like(g))
    dl = slope[:, None] * (hot - p) / temp
    edl = ((eslope[:, None] + 4 * U * slope.abs()[:, None]) * (hot + p) + slope.abs()[:, None] * p * (ee + es[:, None])) / temp
    edl = edl + half_step(dtype) * (dl.abs() + edl) + 1e-37
    return {"loss": (loss, eloss), "logp": (torch.where(on, logp, torch.zeros_like(logp)), elog), "dlogits": (dl, edl),
            "near": near & on}


def newton_schulz(u, steps=5):
    """The iteration as it is written, in u's own type."""
    x = u / (torch.linalg.matrix_norm(u.double(), keepdim=True).to(u.dtype) + 1e-7)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        y = x @ x.mT
        x = 3.4445 * x + (-4.7750 * y + 2.0315 * (y @ y)) @ x
    return x.mT if tall else x


def check(name, got, ref):
    value, bound = ref
    got = got.double()
    assert got.shape == value.shape, name
    same = (got == value) | ((got - value).abs() <= bound)
    if not bool(same.all()):
        off = torch.where(same, torch.zeros_like(got), (got - value).abs() / bound)
        at = int(off.nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{name}: {int((~same).sum())} of {same.numel()} beyond the bound, worst {float(off.flatten()[at]):.3g} "
                             f"times it, at {at}: {float(got.flatten()[at]):.9g} for {float(value.flatten()[at]):.9g}")
