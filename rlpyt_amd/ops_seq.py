"""Operators that train and run a recurrent policy over long sequences and large action sets, as wrappers over
the C ABI (``include/rlpyt_hip.h``); ``rlpyt_amd.ops`` offers them with the others:

* ``gated_scan`` / ``gated_scan_step``: a gated linear recurrence, the parallel counterpart of
  ``lstm_sequence_train`` / ``LstmStep``;
* ``policy_kl_loss`` / ``action_logp``: the clipped policy loss with a KL term straight from logits, next to
  ``ppo_loss``, which takes probabilities of a few actions;
* ``orthogonalize``: the Newton-Schulz products behind ``rlpyt_amd.optim.Muon``.

Arguments that do not fit raise ``ValueError`` before anything is launched, tensors with a forward-mode derivative
(``torch.autograd.forward_ad``) among them.  Kernels run on the current stream of the
tensors' device; workspaces come from torch's allocator per call, so that captured graphs do not share them.  Behind the
checks, the first four run in a small extension (``csrc/seqops.cpp``, loaded by the first call): allocations, launches and autograd
nodes.

Small calls wait for autograd's device thread longer than for the device: a program with one GPU may run its backward passes
under ``torch.autograd.set_multithreading_enabled(False)``, which halves a small scan's time.

A backward pass that is captured into a graph needs what all of torch's autograd needs there: warm up on a side stream, and
drop eager results that still hang on the same leaves (their nodes belong to the other stream; an operator whose own
input is such a leaf raises ``RuntimeError``, in its captured forward pass already; without a backward pass it is captured under
``torch.no_grad()``).
"""
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib

class _Unloaded:
    """Stands in for the extension until the first call that needs it: what does without these operators does without the file."""

    def __getattr__(self, name):
        global _seqops
        try:
            from . import _seqops as loaded   # (after _lib: it takes the C entry points from the library that is loaded there)
        except ImportError as e:
            raise _lib.HipExtensionMissing(
                f"rlpyt_amd/_seqops.so cannot be loaded ({e}). Run `python -c 'import __graft_entry__ as g; g.build()'` (or "
                "`make -C rlpyt_amd/csrc`).") from e
        if loaded.abi_version != _lib.ABI_VERSION:
            raise _lib.HipExtensionMissing(
                f"rlpyt_amd/_seqops.so has ABI {loaded.abi_version}, binding expects {_lib.ABI_VERSION}: rebuild.")
        _seqops = loaded
        return getattr(loaded, name)


_seqops = _Unloaded()

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = (torch.float32, torch.float64, torch.bfloat16, torch.float16)
_BYTES = (torch.bool, torch.uint8)


def _refuse(text):
    raise ValueError(text)


def _need_device(name, first, *others):
    if not first.is_cuda:
        _lib.require_gpu()
        _refuse(f"{name}: tensors on the device are needed, got {first.device}")
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            _refuse(f"{name}: tensors on one device are needed, got {device} and {t.device}")


def _no_tangents(name, *tensors):
    """The kernels see values only: a forward-mode derivative would be lost without a word.  (Tangents live within a level.)"""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            _refuse(f"{name}: forward-mode derivatives are not supported")


# --------------------------------------------------------------------------------------
# gated linear recurrence
# --------------------------------------------------------------------------------------
def _reset_bytes(reset):
    return (reset if reset.dtype in _BYTES else reset != 0).contiguous()


def gated_scan(x, gate, h0=None, reset=None, lengths=None):
    """Gated linear recurrence over ``x, gate [T, B, D]``, all time steps at once::

        z_t = sigmoid(gate_t)        h_t = (1 - z_t) * h_{t-1} + z_t * x_t

    Returns ``(h [T, B, D], hn [B, D])``: every state in the type of ``x``, and the last one in float32.
    Differentiable w.r.t. ``x``, ``gate`` and ``h0`` (once).

    ``x, gate``: float32, bfloat16 or float16, any strides along time and batch (a ``[B, T, D]`` tensor goes
    in as its ``transpose(0, 1)``, the halves of one projection as its ``chunk(2, -1)``); up to 2^28 channels ``B D``
    and less than 2^30 steps.
    ``h0 [B, D]``: the state before the first step (None: 0); other floating types are converted to float32.
    ``reset [T, B]`` (bool, uint8 or nonzero float, as ``done``): the state is cleared BEFORE step t, whatever it
    held.  ``lengths [B]`` (integers, clamped to 0 .. T): steps from ``lengths[b]`` on are not part of sequence b:
    their ``x``, ``gate`` and incoming gradients are not used, their ``h`` and gradients are 0, and ``hn`` is
    the state behind the last step that is (``h0`` for a length of 0).

    States, sums and products are float32, also between the steps of a bfloat16 sequence."""
    if x.dim() != 3 or x.shape != gate.shape:
        _refuse(f"gated_scan: x and gate [T, B, D] are needed, got {tuple(x.shape)} and {tuple(gate.shape)}")
    T, B, D = x.shape
    if T >= 1 << 30 or B * D > 1 << 28:
        _refuse(f"gated_scan: less than 2^30 steps and up to 2^28 channels are supported, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        _refuse(f"gated_scan: x and gate of one type, float32, bfloat16 or float16, are needed, got {x.dtype} "
                f"and {gate.dtype}")
    if h0 is not None and (h0.shape != (B, D) or h0.dtype not in _FLOATS):
        _refuse(f"gated_scan: h0 has to be [B, D] and floating, got {tuple(h0.shape)} {h0.dtype}")
    if reset is not None and (reset.shape != (T, B) or reset.is_complex()):
        _refuse(f"gated_scan: reset has to be [T, B], got {tuple(reset.shape)}")
    if lengths is not None and (lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        _refuse(f"gated_scan: lengths has to be [B], int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")
    _no_tangents("gated_scan", x, gate, h0)
    _need_device("gated_scan", x, gate, h0, reset, lengths)
    if x.numel() == 0:
        hn = torch.zeros((B, D), dtype=torch.float32, device=x.device) if h0 is None else h0.float()
        return x + gate, hn + 0.
    if reset is not None:
        reset = _reset_bytes(reset)
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    if D != 1:
        if x.stride(-1) != 1:
            x = x.contiguous()
        if gate.stride(-1) != 1:
            gate = gate.contiguous()
    return _seqops.gated_scan(x, gate, h0, reset, lengths)


def gated_scan_step(x, gate, state, reset=None):
    """One step of ``gated_scan`` for a sampler or a server: ``x, gate [B, D]``, ``state [B, D]`` float32,
    dense, UPDATED IN PLACE; ``reset [B]`` clears a row's state first.  Returns the new state in the type of
    ``x``.  One launch; not differentiable."""
    shape = x.shape
    if len(shape) != 2 or gate.shape != shape:
        _refuse(f"gated_scan_step: x and gate [B, D] are needed, got {tuple(shape)} and {tuple(gate.shape)}")
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        _refuse(f"gated_scan_step: x and gate of one type, float32, bfloat16 or float16, are needed, got {x.dtype} "
                f"and {gate.dtype}")
    if shape[0] * shape[1] > 1 << 28:
        _refuse(f"gated_scan_step: up to 2^28 channels are supported, got {tuple(shape)}")
    if state.shape != shape or state.dtype != torch.float32 or not state.is_contiguous():
        _refuse("gated_scan_step: state has to be a dense float32 [B, D]")
    if reset is not None and reset.shape != shape[:1]:
        _refuse(f"gated_scan_step: reset has to be [B], got {tuple(reset.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad):
        _refuse("gated_scan_step: not differentiable; call gated_scan, or this under torch.no_grad()")
    _no_tangents("gated_scan_step", x, gate, state)
    _need_device("gated_scan_step", x, gate, state, reset)
    if reset is not None and not (reset.dtype in _BYTES and reset.is_contiguous()):
        reset = _reset_bytes(reset)
    if shape[1] != 1:
        if x.stride(-1) != 1:
            x = x.contiguous()
        if gate.stride(-1) != 1:
            gate = gate.contiguous()
    return _seqops.gated_scan_step(x, gate, state, reset)


# --------------------------------------------------------------------------------------
# clipped policy loss with a KL term, on logits
# --------------------------------------------------------------------------------------
def _logit_rows(name, logits, action):
    """The rows ``[N, V]`` of ``logits [..., V]`` with unit stride along V (a view where the strides allow one), and the
    flat int64 actions."""
    if logits.dim() < 1 or not 0 < logits.shape[-1] <= 1 << 30 or logits.dtype not in _DTYPES:
        _refuse(f"{name}: logits [..., V] in float32, bfloat16 or float16 are needed, got {tuple(logits.shape)} "
                f"{logits.dtype}")
    if action.shape != logits.shape[:-1] or action.is_floating_point() or action.dtype == torch.bool:
        _refuse(f"{name}: one whole action per row of logits is needed, got {tuple(action.shape)} {action.dtype}")
    _need_device(name, logits, action)
    rows = logits.detach()
    if rows.dim() != 2:
        rows = rows.reshape(-1, rows.shape[-1])
    if rows.stride(-1) != 1 and rows.shape[-1] != 1:
        rows = rows.contiguous()
    if action.dtype != torch.int64 or not action.is_contiguous():
        action = action.to(torch.int64).contiguous()
    return rows, action


def _numbers(t):
    """Dense float32, in the order of the rows."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def policy_kl_loss(logits, action, old_logp, advantage, ref_logp=None, valid=None, clip_low=0.2, clip_high=0.2,
                   kl_coeff=0., entropy_coeff=0., grad_scale=1.):
    """Clipped policy loss with a KL term and an entropy bonus over ``softmax(logits)``, as one fused forward
    and backward pass over the logits::

        r = exp(logp - old_logp)      d = ref_logp - logp      kl = exp(d) - d - 1
        loss = mean_valid(-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coeff kl - entropy_coeff H)

    ``logits [..., V]`` float32, bfloat16 or float16, any row stride; ``action [...]`` whole numbers;
    ``old_logp, advantage, ref_logp [...]`` (the log-probabilities as ``action_logp`` gives them) and ``valid
    [...]`` (weights, or a mask) are taken as float32 and as constants.  ``mean_valid`` divides by the sum of ``valid``, of
    either sign; a sum of 0 gives 0.

    Returns ``(loss, scalars)``: ``loss`` is differentiable w.r.t. ``logits`` (one backward pass a call: the
    gradient comes out of the forward pass, is scaled in place and handed on), ``scalars = [loss, pi_loss, kl,
    entropy, clipped share]`` (detached).

    The gradient is rounded to the type of ``logits`` in the forward pass, for an incoming gradient of ``grad_scale``;
    another one costs a pass over it, and a second rounding where their ratio is no power of two.  A loss that is scaled
    against float16's underflow (``(S * loss).backward()``) needs ``grad_scale=S``.

    Logits of -inf are actions that are not allowed.  Rows whose ``valid`` is 0 are not read and have a zero
    gradient, also where their action is out of range; nothing valid gives a loss of 0.  A row that allows
    no action adds 0 and has a zero gradient, but counts in the mean.  In a valid row an action outside 0 .. V-1 or a NaN
    logit makes the loss NaN.  The kl of an action that is not allowed is infinite, and so is a loss with a KL term; the
    row's gradient is NaN then.  With ``kl_coeff`` = 0 a reference policy is watched only: ``scalars`` has its kl, the loss and
    the gradient have nothing of it."""
    lead = logits.shape[:-1]
    for name, t in (("old_logp", old_logp), ("advantage", advantage), ("ref_logp", ref_logp), ("valid", valid)):
        if t is None and name in ("ref_logp", "valid"):
            continue
        if t.shape != lead or t.is_complex():
            _refuse(f"policy_kl_loss: {name} has to be {tuple(lead)}, one number per row of logits, got {tuple(t.shape)}")
    if not (0. <= clip_low <= 1. and clip_high >= 0.):
        _refuse("policy_kl_loss: 0 <= clip_low <= 1 and 0 <= clip_high are needed")
    if ref_logp is None and kl_coeff != 0.:
        _refuse("policy_kl_loss: kl_coeff needs ref_logp")
    if not 0. < grad_scale < float("inf"):
        _refuse("policy_kl_loss: a positive grad_scale is needed")
    _no_tangents("policy_kl_loss", logits, old_logp, advantage, ref_logp, valid)
    rows, action = _logit_rows("policy_kl_loss", logits, action)
    _need_device("policy_kl_loss", rows, old_logp, advantage, ref_logp, valid)
    seed = _unit_seeds.get(logits.device)
    return _seqops.policy_kl_loss(logits, rows, action, _numbers(old_logp), _numbers(advantage), _numbers(ref_logp),
                                  _numbers(valid), clip_low, clip_high, kl_coeff, entropy_coeff, grad_scale,
                                  0 if seed is None else seed.data_ptr())


def action_logp(logits, action):
    """``(log softmax(logits)[action], entropy)``, float32, of every row of ``logits [..., V]`` (float32,
    bfloat16 or float16): what ``policy_kl_loss`` takes as ``old_logp`` and ``ref_logp``.  Reads the logits once.
    A row of -inf only gives ``(-inf, 0)``, an action outside 0 .. V-1 NaN.  Not differentiable: logits that require a
    gradient are taken under ``torch.no_grad()`` only."""
    _no_tangents("action_logp", logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        _refuse("action_logp: not differentiable; call it under torch.no_grad() or with logits.detach()")
    rows, action = _logit_rows("action_logp", logits, action)
    return _seqops.action_logp(logits, rows, action)


# --------------------------------------------------------------------------------------
# orthogonalisation
# --------------------------------------------------------------------------------------
NS_COEFFS = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def _check_polynomial(steps, a, b, c):
    """The library's own check of the polynomial, which comes before the matrices: here an empty one."""
    none, pointer = (ctypes.c_int64 * 1)(0), (ctypes.c_void_p * 1)(None)
    if lib.rlpyt_orthogonalize(0, pointer, none, pointer, none, none, 1, steps, a, b, c, 0., None, None):
        raise _lib.HipArgumentError(_lib.last_error())


def orthogonalize(mats, steps=5, coeffs=NS_COEFFS, eps=1e-7):
    """Newton-Schulz orthogonalisation of an update: ``X = G / (|G|_F + eps)``, then ``steps`` times ``X <-
    a X + (b A + c A A) X`` with ``A = X X^T`` (of the wide form), which moves the singular values towards 1 and keeps
    the singular vectors.

    ``mats``: a tensor ``[..., m, n]`` or a list of such, float32, bfloat16 or float16; returned are new
    dense tensors of the same shapes and types.  All matrices of one type go through the same few launches.  Products
    have 22 bits and float32 sums whatever the type.  Entries below ``2^-37 |G|_F`` are lost, a zero matrix stays zero.
    ``coeffs`` have to keep singular values of 0 .. 1 bounded (below sqrt(8) on the way).  Not differentiable: matrices that
    require a gradient are taken under ``torch.no_grad()`` only."""
    single = isinstance(mats, torch.Tensor)
    mats = [mats] if single else list(mats)
    if not 1 <= steps <= 100 or int(steps) != steps:
        _refuse(f"orthogonalize: 1 to 100 steps are needed, got {steps}")
    if len(coeffs) != 3:
        _refuse("orthogonalize: three coefficients are needed")
    if not eps >= 0.:
        _refuse("orthogonalize: eps >= 0 is needed")
    steps, coeffs = int(steps), [float(v) for v in coeffs]
    _check_polynomial(steps, *coeffs)
    for g in mats:
        if g.dim() < 2 or g.dtype not in _DTYPES:
            _refuse(f"orthogonalize: matrices in float32, bfloat16 or float16 are needed, got {tuple(g.shape)} {g.dtype}")
        if max(g.shape[-2:]) > 1 << 16:
            _refuse(f"orthogonalize: sides up to 65536 are supported, got {tuple(g.shape)}")
    if not mats:
        return []
    _no_tangents("orthogonalize", *mats)
    if torch.is_grad_enabled() and any(g.requires_grad for g in mats):
        _refuse("orthogonalize: not differentiable; call it under torch.no_grad() or with detached matrices")
    _need_device("orthogonalize", *mats)
    device = mats[0].device
    outs, tables = [], {}
    for g in mats:
        o = torch.empty(g.shape, dtype=g.dtype, device=device)
        outs.append(o)
        if g.numel() == 0:
            continue
        table = tables.setdefault(g.dtype, ([], []))
        m, n = g.shape[-2:]
        flat = g.detach()
        if flat.dim() != 3:
            flat = flat.reshape(-1, m, n) if flat.dim() > 3 else flat.unsqueeze(0)
        if flat.stride(-1) != 1 and n != 1:
            flat = flat.contiguous()
        table[1].append(flat)
        size = flat.element_size()
        src, dst, ld, step = flat.data_ptr(), o.data_ptr(), flat.stride(1), flat.stride(0) * size
        for k in range(flat.shape[0]):
            table[0].append((src + k * step, ld, dst + k * m * n * size, m, n))
    for dtype, (table, _) in tables.items():
        k = len(table)
        ins, lds, dsts, rows, cols = zip(*table)
        ins, dsts = (ctypes.c_void_p * k)(*ins), (ctypes.c_void_p * k)(*dsts)
        lds, rows, cols = ((ctypes.c_int64 * k)(*v) for v in (lds, rows, cols))
        ws = torch.empty(lib.rlpyt_orthogonalize_workspace_bytes(rows, cols, k), dtype=torch.uint8, device=device)
        with torch.cuda.device(device):
            check(lib.rlpyt_orthogonalize(_DTYPES[dtype], ins, lds, dsts, rows, cols, k, steps, *coeffs,
                                          float(eps), ws.data_ptr(), torch.cuda.current_stream().cuda_stream),
                  "rlpyt_orthogonalize")
    return outs[0] if single else outs


from .ops import _unit_seeds  # noqa: E402  (ops imports this module at its end)
