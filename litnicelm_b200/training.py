"""Operators of a training step on torch tensors, beside those of the plugin table (section 4 of
include/litnice_backend_b200.h; the kernels are in csrc/train_attention*.cu, csrc/policy_loss.cu and csrc/orthogonal*.cu).

* ``attention_forward`` / ``attention_backward``: attention that keeps one number per row and computes the probabilities
  again in its backward pass, instead of the table's softmax over kept scores.
* ``policy_loss``: clipped policy loss with a KL term and the gradient of the logits, beside ``cross_entropy_mean``.
* ``orthogonalise`` / ``muon_step``: orthogonalised momentum, beside ``adamw_step``.

Tensors are CUDA tensors of one device; views of any strides are taken as they are. Work is enqueued on torch's current
stream of that device, nothing is synchronised, and calls may be captured into a CUDA graph. Workspaces come from torch's allocator
for the call. Tensors that another stream uses need its ordering, as everywhere in torch.

The gradients are explicit, as in the table: nothing here joins torch's autograd, and tensors that would need it are refused
while it records; so are tensors with a tangent of forward mode, and views whose values lie negated in memory (``x.conj().imag``).
Results that are given count as changed in place, as autograd's checks of saved tensors want. There is no fallback: without the library or without a GPU every call raises.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .plugin import NativeError, load_library

_VIEW, _ADDRESS = struct.Struct("<IIQI4x4q12q"), struct.Struct("<Q")  # BackendTensorView, its address 8 bytes in
_KINDS = {torch.float32: 0, torch.int32: 1, torch.bfloat16: 2}


class AttentionOptions(C.Structure):
    _fields_ = [("scale", C.c_float), ("causal", C.c_int32), ("first", C.c_int32), ("window", C.c_int32),
                ("lengths", C.c_void_p)]


class PolicyOptions(C.Structure):
    _fields_ = [("temp", C.c_float), ("clip_low", C.c_float), ("clip_high", C.c_float), ("kl_weight", C.c_float)]


class MuonOptions(C.Structure):
    _fields_ = [("lr", C.c_float), ("mu", C.c_float), ("weight_decay", C.c_float), ("nesterov", C.c_int32),
                ("steps", C.c_int32)]


_lib = None
_GRAD_REFUSED = " requires a gradient: the operators here have explicit backward calls (use torch.no_grad() or detach())"
_PAD = tuple((0,) * (6 - rank) for rank in range(7))
# what torch.cuda.current_stream(index).cuda_stream and torch.cuda.current_device() say, without the objects around it: a
# quarter of the host's time in a small call
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _library():
    global _lib
    if _lib is None:
        lib = load_library()
        P, U = C.c_void_p, C.c_uint64
        for name, args in (("attention_forward", [P] * 7 + [U, P]), ("attention_backward", [P] * 11 + [U, P]),
                           ("policy_loss", [P] * 11 + [U, P]), ("orthogonalise", [P, P, C.c_int32, P, U, P]),
                           ("muon_step", [P] * 5 + [U, P])):
            fn = getattr(lib, "litnice_b200_" + name)
            fn.argtypes, fn.restype = args, C.c_int
        for name, args in (("attention_forward", [P, P]), ("attention_backward", [P, P]), ("policy_loss", [P]),
                           ("orthogonalise", [P])):
            fn = getattr(lib, f"litnice_b200_{name}_workspace")
            fn.argtypes, fn.restype = args, U
        lib.litnice_b200_last_error.argtypes, lib.litnice_b200_last_error.restype = [P], C.c_char_p
        _lib = lib
    return _lib


def _error(rc: int) -> Exception:
    text = _library().litnice_b200_last_error(None).decode()
    return ValueError(text) if rc == -1 else NativeError(f"{text} ({rc})")


def _tensor(t, name: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is not a tensor")


def _plain(t: torch.Tensor, name: str):
    """That the tensor's memory is all there is to it."""
    if t.is_neg():
        raise ValueError(f"{name} is a view of negated values: use resolve_neg()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent: the operators here have no forward-mode derivative")


def _changed(*results):
    """Memory that the caller has given was written."""
    given = [t for t in results if t is not None]
    if given:
        torch.autograd.graph.increment_version(given)


@functools.lru_cache(maxsize=4096)
def _view_head(dtype, shape, strides, name) -> bytes:
    """A view without its address."""
    kind, rank = _KINDS.get(dtype), len(shape)
    if kind is None:
        raise TypeError(f"{name} has type {dtype}")
    if rank > 6:
        raise ValueError(f"{name} has {rank} axes")
    size = 2 if dtype is torch.bfloat16 else 4
    # (rows, cols and their strides repeat the axes; these entries read the axes)
    return _VIEW.pack(1, kind, 0, rank, 0, 0, 0, 0, *shape, *_PAD[rank], *[x * size for x in strides], *_PAD[rank])


def _views(names, tensors):
    """(addresses of the tensors' views, the memory that holds them), checked to be CUDA tensors of one device that autograd does
    not record."""
    recording, device, heads, at, dual = torch.is_grad_enabled(), None, [], 8, forward_ad._current_level >= 0
    for name, t in zip(names, tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} is not a tensor")
        if dual or t.is_neg():
            _plain(t, name)
        if t.device != device:
            if device is not None:
                raise ValueError(f"{name} is on {t.device}, not on {device}")
            device = t.device
            if device.type != "cuda":
                raise ValueError(f"{name} is not a CUDA tensor")
        if recording and t.requires_grad:
            raise ValueError(name + _GRAD_REFUSED)
        heads.append(_view_head(t.dtype, t.shape, t.stride(), name))
    raw = bytearray().join(heads)
    for t in tensors:
        _ADDRESS.pack_into(raw, at, t.data_ptr())
        at += 152
    held = (C.c_char * len(raw)).from_buffer(raw)
    base = C.addressof(held)
    return range(base, base + len(raw), 152), held


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _run(device: torch.device, fn, *args):
    """The entry point on the current stream of the tensors' device."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise _error(rc)


def _workspace(nbytes: int, device) -> torch.Tensor:
    if nbytes == 0:
        raise _error(-1)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)  # (on a 512-byte boundary)


def _vector(t: Optional[torch.Tensor], name: str, count: int, dtype, device) -> Optional[int]:
    """Address of a dense vector of `count` elements."""
    if t is None:
        return None
    _tensor(t, name)
    if forward_ad._current_level >= 0 or t.is_neg():
        _plain(t, name)
    if t.dtype != dtype or t.shape != (count,) or (count > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a dense {dtype} vector of {count} elements")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(name + _GRAD_REFUSED)
    return t.data_ptr()


def _steps(steps: int) -> int:
    if not 0 <= steps <= 100:  # (before ctypes takes its lowest 32 bits)
        raise ValueError("steps is out of range")
    return steps


def _options(q: torch.Tensor, scale, causal, first, window, lengths) -> AttentionOptions:
    if q.dim() != 4:
        raise ValueError("q must be [streams, rows, heads, dim]")
    if not (0 <= first < 1 << 30 and 0 <= window < 1 << 30):
        raise ValueError("first and window must be at least 0")
    return AttentionOptions(1 / math.sqrt(max(1, q.shape[3])) if scale is None else scale, 1 if causal else 0, first, window,
                            _vector(lengths, "lengths", q.shape[0], torch.int32, q.device))


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True,
                      first: int = 0, window: int = 0, lengths: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [streams, n, heads, dim], lse [streams, heads, n]) of q [streams, n, heads, dim] over k and v [streams, m, groups, dim],
    float32 or bfloat16, dim up to 128; query head h uses key head h * groups // heads.

    Row i stands at position first + i and sees key j if j < m, j < lengths[stream], with ``causal`` j <= first + i, with a
    ``window`` j > first + i - window. A row that sees no key has out 0 and lse -inf. scale: 1 / sqrt(dim) if None."""
    _tensor(q, "q")
    given, out = out, _like(q) if out is None else out
    (vq, vk, vv, vo), held = _views(("q", "k", "v", "out"), (q, k, v, out))
    o = _options(q, scale, causal, first, window, lengths)
    streams, n, heads = q.shape[:3]
    lse = torch.empty((streams, heads, n), dtype=torch.float32, device=q.device)
    lib = _library()
    work = _workspace(lib.litnice_b200_attention_forward_workspace(vq, vk), q.device)
    _run(q.device, lib.litnice_b200_attention_forward, vq, vk, vv, C.addressof(o), vo, lse.data_ptr(), work.data_ptr(), work.numel())
    _changed(given)
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True, first: int = 0, window: int = 0,
                       lengths: Optional[torch.Tensor] = None, dq: Optional[torch.Tensor] = None,
                       dk: Optional[torch.Tensor] = None,
                       dv: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv): gradients of sum(out * dout), from what ``attention_forward`` with the same options returned. Key heads
    shared by query heads receive the sum over those. dq, dk and dv may be given, slices of one buffer for instance. Weights come
    from lse, so they are off by |lse| 2^-24 of themselves: scores far beyond thousands leave the gradients no accuracy."""
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (lse, "lse")):
        _tensor(t, name)
    _plain(lse, "lse")
    given = dq, dk, dv
    dq = _like(q) if dq is None else dq
    dk = _like(k) if dk is None else dk
    dv = _like(v) if dv is None else dv
    (vd, vq, vk, vv, vo, wq, wk, wv), held = _views(("dout", "q", "k", "v", "out", "dq", "dk", "dv"), (dout, q, k, v, out, dq, dk, dv))
    o = _options(q, scale, causal, first, window, lengths)
    streams, n, heads = q.shape[:3]
    if lse.dtype != torch.float32 or lse.shape != (streams, heads, n) or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be what attention_forward returned")
    lib = _library()
    work = _workspace(lib.litnice_b200_attention_backward_workspace(vq, vk), q.device)
    _run(q.device, lib.litnice_b200_attention_backward, vd, vq, vk, vv, vo, lse.data_ptr(), C.addressof(o), wq, wk, wv,
         work.data_ptr(), work.numel())
    _changed(*given)
    return dq, dk, dv


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor, *,
                ref_logp: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, temp: float = 1.0,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_weight: float = 0.0, gradient: bool = True,
                dlogits: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(loss, logp [rows], dlogits) of logits [rows, vocab], float32 or bfloat16 with contiguous columns.

    With z = logits / temp, logp = log_softmax(z)[target], r = exp(logp - old_logp), d = ref_logp - logp:
    loss = sum weight (-min(r advantage, clip(r, 1 - clip_low, 1 + clip_high) advantage) + kl_weight (exp d - d - 1)) / sum weight.
    Rows of weight 0 are not read; their logp and gradient are 0. Weights whose sum is 0 give loss 0 and gradients of 0. A target
    outside the vocabulary in another row gives NaN there and in the loss. dlogits may be given, logits itself included; with
    ``gradient`` false it is None."""
    _tensor(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, vocab]")
    rows, dev, given = logits.shape[0], logits.device, dlogits if gradient else None
    if gradient:
        dlogits = _like(logits) if dlogits is None else dlogits
        (vz, vd), held = _views(("logits", "dlogits"), (logits, dlogits))
    else:
        (vz,), held = _views(("logits",), (logits,))
        vd = dlogits = None
    o = PolicyOptions(temp, clip_low, clip_high, kl_weight)
    loss, logp = torch.empty((), dtype=torch.float32, device=dev), torch.empty(rows, dtype=torch.float32, device=dev)
    lib = _library()
    work = _workspace(lib.litnice_b200_policy_loss_workspace(vz), dev)
    _run(dev, lib.litnice_b200_policy_loss, vz, _vector(targets, "targets", rows, torch.int32, dev),
         _vector(old_logp, "old_logp", rows, torch.float32, dev), _vector(advantage, "advantage", rows, torch.float32, dev),
         _vector(ref_logp, "ref_logp", rows, torch.float32, dev), _vector(weight, "weight", rows, torch.float32, dev),
         C.addressof(o), loss.data_ptr(), logp.data_ptr(), vd, work.data_ptr(), work.numel())
    _changed(given)
    return loss, logp, dlogits


def orthogonalise(x: torch.Tensor, *, steps: int = 5, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every matrix of x [..., m, n] float32 with its singular values driven towards 1: X = x / (|x| + 1e-7), then ``steps`` times
    X <- 3.4445 X + (-4.7750 A + 2.0315 A A) X with A = X X^T (in the smaller side's space). out may be x, with x's strides. But for
    matrices with one side of at most 64 and the other of at most 4096, X and A are held in 22 bits between products summed in 32."""
    _tensor(x, "x")
    given, out = out, _like(x) if out is None else out
    _steps(steps)
    (vx, vo), held = _views(("x", "out"), (x, out))
    lib = _library()
    work = _workspace(lib.litnice_b200_orthogonalise_workspace(vx), x.device)
    _run(x.device, lib.litnice_b200_orthogonalise, vx, vo, steps, work.data_ptr(), work.numel())
    _changed(given)
    return out


def muon_step(params: torch.Tensor, grads: torch.Tensor, momentum: torch.Tensor, lr: float, *, mu: float = 0.95,
              weight_decay: float = 0.0, nesterov: bool = True, steps: int = 5) -> None:
    """One optimiser step on matrices [..., m, n] float32, in place: momentum <- mu momentum + grads, U = grads + mu momentum (or
    momentum without ``nesterov``), params <- (1 - lr weight_decay) params - lr sqrt(max(1, m / n)) orthogonalise(U)."""
    o = MuonOptions(lr, mu, weight_decay, 1 if nesterov else 0, _steps(steps))
    (vp, vg, vm), held = _views(("params", "grads", "momentum"), (params, grads, momentum))
    lib = _library()
    work = _workspace(lib.litnice_b200_orthogonalise_workspace(vg), grads.device)
    _run(grads.device, lib.litnice_b200_muon_step, vp, vg, vm, C.addressof(o), work.data_ptr(), work.numel())
    _changed(params, momentum)
