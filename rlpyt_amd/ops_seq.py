"""Operators that train and run a recurrent policy over long sequences and large action sets, as wrappers over
the C ABI (``include/rlpyt_hip.h``); ``rlpyt_amd.ops`` offers them with the others:

* ``gated_scan`` / ``gated_scan_step``: a gated linear recurrence, the parallel counterpart of
  ``lstm_sequence_train`` / ``LstmStep``;
* ``policy_kl_loss`` / ``action_logp``: the clipped policy loss with a KL term straight from logits, next to
  ``ppo_loss``, which takes probabilities of a few actions;
* ``orthogonalize``: the Newton-Schulz products behind ``rlpyt_amd.optim.Muon``.

Arguments that do not fit raise ``ValueError`` before anything is launched.  Kernels run on the current stream of the
tensors' device; workspaces come from torch's allocator per call, so that captured graphs do not share them.
"""
import ctypes

import torch

from . import _lib
from ._lib import check, lib
from .utils import ktimer

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = (torch.float32, torch.float64, torch.bfloat16, torch.float16)


def _need(cond, text):
    if not cond:
        raise ValueError(text)


def _need_device(name, first, *others):
    _lib.require_gpu()
    _need(first.is_cuda, f"{name}: tensors on the device are needed, got {first.device}")
    for t in others:
        _need(t is None or t.device == first.device,
              f"{name}: tensors on one device are needed, got {first.device} and {getattr(t, 'device', None)}")


def _p(t):
    return None if t is None else t.data_ptr()


class _on:
    """The device of ``t`` as the current one; ``as`` gives its current stream."""
    __slots__ = ("index", "before")

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _bytes(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


# --------------------------------------------------------------------------------------
# gated linear recurrence
# --------------------------------------------------------------------------------------
def _unit_rows(t):
    """``t`` with unit stride along its last axis."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like_rows(x):
    """An empty ``[T, B, D]`` whose rows lie in memory in the order of ``x``'s: time or batch first."""
    T, B, D = x.shape
    if T > 1 and B > 1 and x.stride(1) > x.stride(0):
        return torch.empty((B, T, D), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((T, B, D), dtype=x.dtype, device=x.device)


def _scan_forward(x, gate, h0, reset, lengths, keep):
    T, B, D = x.shape
    h = _like_rows(x)
    hn = torch.empty((B, D), dtype=torch.float32, device=x.device)
    states = (torch.empty((lib.rlpyt_gated_scan_state_rows(T), B, D), dtype=torch.float32, device=x.device)
              if keep else None)
    ws = _bytes(lib.rlpyt_gated_scan_workspace_bytes(T, B, D), x)
    with _on(x) as stream, ktimer.region("gated_scan", 3 * x.numel() * x.element_size()):
        check(lib.rlpyt_gated_scan_fwd(
            _DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0),
            gate.stride(1), _p(h0), _p(reset), _p(lengths), h.data_ptr(), h.stride(0), h.stride(1),
            hn.data_ptr(), _p(states), T, B, D, _p(ws), stream), "rlpyt_gated_scan_fwd")
    return h, hn, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, reset, lengths):
        h0f = None if h0 is None else h0.detach().to(torch.float32).contiguous()
        h, hn, states = _scan_forward(x, gate, h0f, reset, lengths, True)
        ctx.save_for_backward(x, gate, reset, lengths, states)
        ctx.h0_dtype = None if h0 is None else h0.dtype
        ctx.set_materialize_grads(False)
        return h, hn

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dhn):
        x, gate, reset, lengths, states = ctx.saved_tensors
        if dh is None and dhn is None:
            return None, None, None, None, None
        T, B, D = x.shape
        if dh is None:
            dh = torch.zeros(D, dtype=x.dtype, device=x.device).expand(T, B, D)
        dh = _unit_rows(dh.to(x.dtype))
        dhn = None if dhn is None else dhn.to(torch.float32).contiguous()
        dx, dgate = _like_rows(x), _like_rows(x)
        dh0 = (torch.empty((B, D), dtype=torch.float32, device=x.device)
               if ctx.h0_dtype is not None and ctx.needs_input_grad[2] else None)
        ws = _bytes(lib.rlpyt_gated_scan_workspace_bytes(T, B, D), x)
        with _on(x) as stream, ktimer.region("gated_scan_bwd", 5 * x.numel() * x.element_size()):
            check(lib.rlpyt_gated_scan_bwd(
                _DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0),
                gate.stride(1), dh.data_ptr(), dh.stride(0), dh.stride(1), _p(dhn), _p(reset), _p(lengths),
                states.data_ptr(), dx.data_ptr(), dx.stride(0), dx.stride(1), dgate.data_ptr(), dgate.stride(0),
                dgate.stride(1), _p(dh0), T, B, D, _p(ws), stream), "rlpyt_gated_scan_bwd")
        return dx, dgate, None if dh0 is None else dh0.to(ctx.h0_dtype), None, None


def gated_scan(x, gate, h0=None, reset=None, lengths=None):
    """Gated linear recurrence over ``x, gate [T, B, D]``, all time steps at once::

        z_t = sigmoid(gate_t)        h_t = (1 - z_t) * h_{t-1} + z_t * x_t

    Returns ``(h [T, B, D], hn [B, D])``: every state in the type of ``x``, and the last one in float32.
    Differentiable w.r.t. ``x``, ``gate`` and ``h0`` (once).

    ``x, gate``: float32, bfloat16 or float16, any strides along time and batch (a ``[B, T, D]`` tensor goes
    in as its ``transpose(0, 1)``, the halves of one projection as its ``chunk(2, -1)``).
    ``h0 [B, D]``: the state before the first step (None: 0); a bfloat16 or float16 one is widened.
    ``reset [T, B]`` (bool, uint8 or nonzero float, as ``done``): the state is cleared BEFORE step t, whatever it
    held.  ``lengths [B]`` (integers, clamped to 0 .. T): steps from ``lengths[b]`` on are not part of sequence b:
    their ``x``, ``gate`` and incoming gradients are not used, their ``h`` and gradients are 0, and ``hn`` is
    the state behind the last step that is (``h0`` for a length of 0).

    States, sums and products are float32, also between the steps of a bfloat16 sequence."""
    _need(x.dim() == 3 and x.shape == gate.shape,
          f"gated_scan: x and gate [T, B, D] are needed, got {tuple(x.shape)} and {tuple(gate.shape)}")
    T, B, D = x.shape
    _need(x.dtype in _DTYPES and gate.dtype == x.dtype,
          f"gated_scan: x and gate of one type, float32, bfloat16 or float16, are needed, got {x.dtype} and {gate.dtype}")
    _need(h0 is None or (h0.shape == (B, D) and h0.dtype in _FLOATS),
          "gated_scan: h0 has to be [B, D] and floating")
    _need(reset is None or (reset.shape == (T, B) and not reset.is_complex()), "gated_scan: reset has to be [T, B]")
    _need(lengths is None or (lengths.shape == (B,) and lengths.dtype in (torch.int32, torch.int64)),
          "gated_scan: lengths has to be [B], int32 or int64")
    _need_device("gated_scan", x, gate, h0, reset, lengths)
    if x.numel() == 0:
        hn = torch.zeros((B, D), dtype=torch.float32, device=x.device) if h0 is None else h0.float()
        return x + gate, hn + 0.
    if reset is not None:
        reset = (reset if reset.dtype in (torch.bool, torch.uint8) else reset != 0).contiguous().view(torch.uint8)
    if lengths is not None:
        lengths = lengths.to(torch.int64).contiguous()
    x, gate = _unit_rows(x), _unit_rows(gate)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, h0, reset, lengths)
    h0 = None if h0 is None else h0.detach().to(torch.float32).contiguous()
    return _scan_forward(x.detach(), gate.detach(), h0, reset, lengths, False)[:2]


def gated_scan_step(x, gate, state, reset=None):
    """One step of ``gated_scan`` for a sampler or a server: ``x, gate [B, D]``, ``state [B, D]`` float32,
    dense, UPDATED IN PLACE; ``reset [B]`` clears a row's state first.  Returns the new state in the type of
    ``x``.  One launch; not differentiable."""
    _need(x.dim() == 2 and x.shape == gate.shape,
          f"gated_scan_step: x and gate [B, D] are needed, got {tuple(x.shape)} and {tuple(gate.shape)}")
    _need(x.dtype in _DTYPES and gate.dtype == x.dtype,
          f"gated_scan_step: x and gate of one type, float32, bfloat16 or float16, are needed, got {x.dtype} and {gate.dtype}")
    _need(state.shape == x.shape and state.dtype == torch.float32 and state.is_contiguous(),
          "gated_scan_step: state has to be a dense float32 [B, D]")
    _need(reset is None or reset.shape == x.shape[:1], "gated_scan_step: reset has to be [B]")
    _need(not (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad)),
          "gated_scan_step: not differentiable; call gated_scan, or this under torch.no_grad()")
    _need_device("gated_scan_step", x, gate, state, reset)
    if reset is not None:
        reset = (reset if reset.dtype in (torch.bool, torch.uint8) else reset != 0).contiguous()
    x, gate = _unit_rows(x), _unit_rows(gate)
    B, D = x.shape
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    with _on(x) as stream:
        check(lib.rlpyt_gated_scan_step(_DTYPES[x.dtype], x.data_ptr(), x.stride(0), gate.data_ptr(),
                                        gate.stride(0), _p(reset), state.data_ptr(), y.data_ptr(), B, D, stream),
              "rlpyt_gated_scan_step")
    torch.autograd.graph.increment_version([state])   # written through a raw pointer
    return y


# --------------------------------------------------------------------------------------
# clipped policy loss with a KL term, on logits
# --------------------------------------------------------------------------------------
def _logit_rows(name, logits, action):
    _need(logits.dim() >= 1 and logits.shape[-1] > 0 and logits.dtype in _DTYPES,
          f"{name}: logits [..., V] in float32, bfloat16 or float16 are needed, got {tuple(logits.shape)} {logits.dtype}")
    _need(action.shape == logits.shape[:-1] and not action.is_floating_point() and action.dtype != torch.bool,
          f"{name}: one whole action per row of logits is needed, got {tuple(action.shape)} {action.dtype}")


def _flat_rows(logits):
    """``[..., V]`` -> ``[N, V]`` with unit stride along V (a view where the strides allow one)."""
    return _unit_rows(logits.detach().reshape(-1, logits.shape[-1]))


class _PolicyKlLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, action, old_logp, advantage, ref_logp, valid, clip_low, clip_high, kl_coeff,
                entropy_coeff, needs_grad):
        rows = _flat_rows(logits)
        N, V = rows.shape
        code = _DTYPES[rows.dtype]
        scalars = torch.empty(5, dtype=torch.float32, device=rows.device)
        grad = torch.empty((N, V), dtype=rows.dtype, device=rows.device) if needs_grad else None
        ws = _bytes(lib.rlpyt_policy_loss_workspace_bytes(code, N, V), rows)
        with _on(rows) as stream, ktimer.region("policy_kl_loss", (1 + needs_grad) * rows.numel() * rows.element_size()):
            check(lib.rlpyt_policy_kl_loss_fwd_bwd(
                code, rows.data_ptr(), rows.stride(0), action.data_ptr(), old_logp.data_ptr(),
                advantage.data_ptr(), _p(ref_logp), _p(valid), N, V, clip_low, clip_high, kl_coeff,
                entropy_coeff, scalars.data_ptr(), None, None, _p(grad), ws.data_ptr(), stream),
                "rlpyt_policy_kl_loss_fwd_bwd")
        ctx.grad, ctx.shape = grad, logits.shape
        ctx.mark_non_differentiable(scalars)
        return scalars[0], scalars

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_scalars):
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            raise RuntimeError("policy_kl_loss: its gradient went out with the first backward pass (it is scaled in "
                               "place); run the loss again")
        from .ops import _is_unit_seed
        if not _is_unit_seed(g_loss):
            with _on(grad) as stream:
                check(lib.rlpyt_scale_unless_one(_DTYPES[grad.dtype], grad.data_ptr(), grad.numel(),
                                                 g_loss.float().data_ptr(), stream), "rlpyt_scale_unless_one")
        return (grad.reshape(ctx.shape),) + (None,) * 10


def policy_kl_loss(logits, action, old_logp, advantage, ref_logp=None, valid=None, clip_low=0.2, clip_high=0.2,
                   kl_coeff=0., entropy_coeff=0.):
    """Clipped policy loss with a KL term and an entropy bonus over ``softmax(logits)``, as one fused forward
    and backward pass over the logits::

        r = exp(logp - old_logp)      d = ref_logp - logp      kl = exp(d) - d - 1
        loss = mean_valid(-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coeff kl - entropy_coeff H)

    ``logits [..., V]`` float32, bfloat16 or float16, any row stride; ``action [...]`` whole numbers;
    ``old_logp, advantage, ref_logp [...]`` (the log-probabilities as ``action_logp`` gives them) and ``valid
    [...]`` (weights, or a mask) are taken as float32.  ``mean_valid`` divides by the sum of ``valid``.

    Returns ``(loss, scalars)``: ``loss`` is differentiable w.r.t. ``logits`` (one backward pass a call: the
    gradient comes out of the forward pass, is scaled in place and handed on), ``scalars = [loss, pi_loss, kl,
    entropy, clipped share]`` (detached).

    Logits of -inf are actions that are not allowed.  Rows whose ``valid`` is 0 are not read and have a zero
    gradient, also where their action is out of range; nothing valid gives a loss of 0.  A row that allows
    no action adds 0 and has a zero gradient, but counts in the mean.  In a valid row an action outside 0 .. V-1 or a NaN
    logit makes the loss NaN; with a KL term, so does the gradient of an action that is not allowed (its kl is infinite)."""
    _logit_rows("policy_kl_loss", logits, action)
    lead = logits.shape[:-1]
    for name, t in (("old_logp", old_logp), ("advantage", advantage), ("ref_logp", ref_logp), ("valid", valid)):
        _need(t is None and name in ("ref_logp", "valid") or t is not None and t.shape == lead and not t.is_complex(),
              f"policy_kl_loss: {name} has to be {tuple(lead)}, one number per row of logits")
    _need(0. <= clip_low <= 1. and clip_high >= 0., "policy_kl_loss: 0 <= clip_low <= 1 and 0 <= clip_high are needed")
    _need(ref_logp is not None or kl_coeff == 0., "policy_kl_loss: kl_coeff needs ref_logp")
    _need_device("policy_kl_loss", logits, action, old_logp, advantage, ref_logp, valid)

    def flat(t):
        return None if t is None else t.detach().to(torch.float32).reshape(-1).contiguous()

    action = action.reshape(-1).to(torch.int64).contiguous()
    needs_grad = torch.is_grad_enabled() and logits.requires_grad
    return _PolicyKlLoss.apply(logits, action, flat(old_logp), flat(advantage), flat(ref_logp), flat(valid),
                               float(clip_low), float(clip_high), float(kl_coeff), float(entropy_coeff), needs_grad)


def action_logp(logits, action):
    """``(log softmax(logits)[action], entropy)``, float32, of every row of ``logits [..., V]`` (float32,
    bfloat16 or float16): what ``policy_kl_loss`` takes as ``old_logp`` and ``ref_logp``.  Reads the logits once; not
    differentiable.  A row of -inf only gives ``(-inf, 0)``, an action outside 0 .. V-1 NaN."""
    _logit_rows("action_logp", logits, action)
    _need_device("action_logp", logits, action)
    rows = _flat_rows(logits)
    N, V = rows.shape
    action = action.reshape(-1).to(torch.int64).contiguous()
    code = _DTYPES[rows.dtype]
    out = torch.empty((2, N), dtype=torch.float32, device=rows.device)
    ws = _bytes(lib.rlpyt_policy_loss_workspace_bytes(code, N, V), rows)
    with _on(rows) as stream, ktimer.region("action_logp", rows.numel() * rows.element_size()):
        check(lib.rlpyt_action_logp(code, rows.data_ptr(), rows.stride(0), action.data_ptr(), N, V,
                                    out[0].data_ptr(), out[1].data_ptr(), ws.data_ptr(), stream),
              "rlpyt_action_logp")
    lead = logits.shape[:-1]
    return out[0].reshape(lead), out[1].reshape(lead)


# --------------------------------------------------------------------------------------
# orthogonalisation
# --------------------------------------------------------------------------------------
NS_COEFFS = (3.4445, -4.7750, 2.0315)


def orthogonalize(mats, steps=5, coeffs=NS_COEFFS, eps=1e-7):
    """Newton-Schulz orthogonalisation of an update: ``X = G / (|G|_F + eps)``, then ``steps`` times ``X <-
    a X + (b A + c A A) X`` with ``A = X X^T`` (of the wide form), which moves the singular values towards 1 and keeps
    the singular vectors.

    ``mats``: a tensor ``[..., m, n]`` or a list of such, float32, bfloat16 or float16; returned are new
    dense tensors of the same shapes and types.  All matrices of one type go through the same few launches.  Products
    have 22 bits and float32 sums whatever the type.  Entries below ``2^-37 |G|_F`` are lost, a zero matrix stays zero.
    ``coeffs`` have to keep singular values of 0 .. 1 bounded (below sqrt(8) on the way).  Not differentiable."""
    single = isinstance(mats, torch.Tensor)
    mats = [mats] if single else list(mats)
    _need(int(steps) == steps and 1 <= steps <= 100, "orthogonalize: 1 to 100 steps are needed")
    _need(len(coeffs) == 3, "orthogonalize: three coefficients are needed")
    _need(eps >= 0., "orthogonalize: eps >= 0 is needed")
    for g in mats:
        _need(g.dim() >= 2 and g.dtype in _DTYPES,
              f"orthogonalize: matrices in float32, bfloat16 or float16 are needed, got {tuple(g.shape)} {g.dtype}")
    if not mats:
        return []
    _need_device("orthogonalize", *mats)
    outs = [torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in mats]
    for dtype, code in _DTYPES.items():
        table, keep = [], []
        for g, o in zip(mats, outs):
            if g.dtype != dtype or g.numel() == 0:
                continue
            m, n = g.shape[-2:]
            flat = _unit_rows(g.detach().reshape(-1, m, n))
            keep.append(flat)
            size, ld = flat.element_size(), flat.stride(1)
            table += [(flat.data_ptr() + k * flat.stride(0) * size, ld, o.data_ptr() + k * m * n * size, m, n)
                      for k in range(flat.shape[0])]
        if not table:
            continue
        k = len(table)
        ins, lds, dsts, rows, cols = zip(*table)
        ins, dsts = (ctypes.c_void_p * k)(*ins), (ctypes.c_void_p * k)(*dsts)
        lds, rows, cols = ((ctypes.c_int64 * k)(*v) for v in (lds, rows, cols))
        ws = _bytes(lib.rlpyt_orthogonalize_workspace_bytes(rows, cols, k), keep[0])
        with _on(keep[0]) as stream, ktimer.region("orthogonalize", 0):
            check(lib.rlpyt_orthogonalize(code, ins, lds, dsts, rows, cols, k, int(steps), *map(float, coeffs),
                                          float(eps), ws.data_ptr(), stream), "rlpyt_orthogonalize")
    return outs[0] if single else outs
