"""The sequence operators on the device against plain implementations in 64 bits.

Tolerances.  Rounding to an output type t is off by at most HALF[t] = finfo(t).eps / 2 of the value.  On top
of it comes what 32-bit arithmetic leaves:
* gated_scan: a step adds at most c 2^-24 max|values| with c = 16 (the exponent of e^-|gate|, |gate| < 8, one
  reciprocal, two products, one sum), and a step's error fades by 1 - z a step: with gates >= -6 at most
  1 / z = 404 steps count.
* policy_kl_loss: e^(x - max) is off by (|x - max| + 4) 2^-24 relative, |x - max| < 64 where it matters; a row's
  sum adds 2^-20 (up to 512 terms a lane, in sequence); log and everything per row is 64 bits.
* orthogonalize: the factors are 22 bits (2^-23 of the row norms), amplified by up to 484 over five
  steps where the singular value is tiny, of which a fraction 1 / sqrt(m) is left relative to the result's norm."""
import copy
import math

import pytest
import torch

from rlpyt_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = (torch.float32, torch.bfloat16, torch.float16)
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------- gated scan
def scan64(x, gate, h0=None, reset=None, lengths=None, dh=None, dhn=None):
    """Forward and backward, one step after the other, by the formulas."""
    T, B, D = x.shape
    x, gate = x.detach().double(), gate.detach().double()
    z, a = torch.sigmoid(gate), torch.sigmoid(-gate)
    live = torch.ones(T, B, 1, dtype=torch.bool, device=x.device)
    if lengths is not None:
        live = (torch.arange(T, device=x.device)[:, None] < lengths).unsqueeze(-1)
    clear = torch.zeros_like(live) if reset is None else reset.bool().unsqueeze(-1)
    zero = torch.zeros(B, D, dtype=torch.float64, device=x.device)
    s = zero if h0 is None else h0.detach().double()
    h, prev = [], []
    for t in range(T):
        k = torch.where(clear[t] & live[t], zero, s)
        prev.append(k)
        s = torch.where(live[t], a[t] * k + z[t] * x[t], s)
        h.append(torch.where(live[t], s, zero))
    out = {"h": torch.stack(h), "hn": s}
    if dh is not None:
        G, dx, dg = (zero if dhn is None else dhn.double()), [], []
        for t in range(T - 1, -1, -1):
            full = G + dh[t].double()
            dx.append(torch.where(live[t], full * z[t], zero))
            dg.append(torch.where(live[t], full * (x[t] - prev[t]) * z[t] * a[t], zero))
            G = torch.where(live[t], torch.where(clear[t], zero, a[t] * full), G)
        out.update(dx=torch.stack(dx[::-1]), dgate=torch.stack(dg[::-1]), dh0=G)
    return out


def scan_close(got, want, T):
    for k, w in want.items():
        g = got[k].double()
        finite = w[torch.isfinite(w)]
        top = float(finite.abs().max()) if finite.numel() else 0.
        if k in ("dx", "dgate"):
            top = max(top, float(want["dh0"].abs().max()), 1.)
        tol = HALF[got[k].dtype] * w.abs() + 16 * min(T, 404) * 2. ** -24 * max(top, 1.)
        tol += torch.finfo(got[k].dtype).tiny
        assert bool(((g - w).abs() <= tol).all()), (k, float((g - w).abs().max()), top)


def scan_data(T, B, D, dtype, seed, reset=False, lengths=False, layout="dense"):
    g = gen(seed)
    if layout == "halves":          # the halves of one projection
        p = torch.randn(T, B, 2 * D, device=DEV, generator=g).to(dtype)
        x, gate = p.chunk(2, -1)
    elif layout == "batch first":
        x, gate = (torch.randn(B, T, D, device=DEV, generator=g).to(dtype).transpose(0, 1) for _ in range(2))
    elif layout == "odd start":     # rows that start at odd elements
        x, gate = (torch.randn(T, B, D + 3, device=DEV, generator=g).to(dtype)[..., 1:D + 1] for _ in range(2))
    elif layout == "columns":       # no unit stride along D
        x, gate = (torch.randn(T, D, B, device=DEV, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    else:
        x, gate = (torch.randn(T, B, D, device=DEV, generator=g).to(dtype) for _ in range(2))
    gate = (gate - 1).clamp(-6, 7) if layout in ("dense", "columns") else gate
    h0, dhn = (torch.randn(B, D, device=DEV, generator=g) for _ in range(2))
    dh = torch.randn(T, B, D, device=DEV, generator=g).to(dtype)
    rs = torch.rand(T, B, device=DEV, generator=g) < 0.1 if reset else None
    ln = torch.randint(0, T + 1, (B,), device=DEV, generator=g) if lengths else None
    if ln is not None:
        ln[0] = T
        ln[-1] = ln[-1] if B < 3 else 0
    return x, gate, h0, dh, dhn, rs, ln


def scan_grads(x, gate, h0, dh, dhn, rs, ln):
    x, gate, h0 = (t.detach().requires_grad_(True) for t in (x, gate, h0))
    h, hn = ops.gated_scan(x, gate, h0, reset=rs, lengths=ln)
    dx, dgate, dh0 = torch.autograd.grad((h, hn), (x, gate, h0), (dh, dhn))
    return {"h": h, "hn": hn, "dx": dx, "dgate": dgate, "dh0": dh0}


SIZES = [(1, 1, 1), (1, 3, 5), (2, 1, 64), (7, 2, 3), (8, 1, 128), (9, 2, 130), (63, 1, 127), (64, 4, 32), (65, 3, 33),
         (85, 4, 512), (129, 300, 70), (257, 2, 70), (1001, 3, 333), (5000, 1, 24)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reset,lengths", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gated_scan(size, reset, lengths, dtype):
    T, B, D = size
    data = scan_data(T, B, D, dtype, 1, reset, lengths)
    x, gate, h0, dh, dhn, rs, ln = data
    got = scan_grads(*data)
    scan_close(got, scan64(x, gate, h0, rs, ln, dh, dhn), T)
    with torch.no_grad():            # the same kernels without what the backward pass needs
        h, hn = ops.gated_scan(x, gate, h0, reset=rs, lengths=ln)
    assert torch.equal(h, got["h"]) and torch.equal(hn, got["hn"])


@pytest.mark.parametrize("layout", ["halves", "batch first", "odd start", "columns"])
@pytest.mark.parametrize("size", [(65, 3, 34), (700, 2, 130), (20, 600, 64)], ids=str)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_gated_scan_strides(size, layout, dtype):
    T, B, D = size
    data = scan_data(T, B, D, dtype, 2, True, True, layout)
    x, gate, h0, dh, dhn, rs, ln = data
    got = scan_grads(*data)
    scan_close(got, scan64(x, gate, h0, rs, ln, dh, dhn), T)
    if layout == "batch first":
        assert got["h"].transpose(0, 1).is_contiguous() and got["dx"].transpose(0, 1).is_contiguous()


def test_gated_scan_segments_and_single_segment_agree_with_64_bits_on_one_long_sequence():
    T, B, D = 20000, 1, 256           # few channels: time is cut into segments
    _lib.variant_reset()
    data = scan_data(T, B, D, torch.float32, 3, True)
    x, gate, h0, dh, dhn, rs, ln = data
    got = scan_grads(*data)
    names = _lib.variant_counts()
    assert any("gated_scan_fwd_kernel" in n and n.endswith("true>") for n in names), names
    scan_close(got, scan64(x, gate, h0, rs, ln, dh, dhn), T)


def test_gated_scan_optional_arguments():
    x, gate, h0, dh, dhn, _, _ = scan_data(40, 3, 17, torch.float32, 4)
    xg, gg = x.clone().requires_grad_(True), gate.clone().requires_grad_(True)
    h, hn = ops.gated_scan(xg, gg)                       # no state: zeros
    want = scan64(x, gate, None, None, None, torch.zeros_like(dh), dhn)
    dx, dgate = torch.autograd.grad(hn, (xg, gg), dhn, retain_graph=True)      # a gradient of the last state only
    scan_close({"h": h, "hn": hn}, {k: want[k] for k in ("h", "hn")}, 40)
    assert torch.allclose(dx.double(), want["dx"], rtol=1e-4, atol=1e-5)
    assert torch.allclose(dgate.double(), want["dgate"], rtol=1e-4, atol=1e-5)
    want = scan64(x, gate, None, None, None, torch.ones_like(dh))
    dx, = torch.autograd.grad(h.sum(), xg)               # an expanded gradient (all strides 0)
    assert torch.allclose(dx.double(), want["dx"], rtol=1e-4, atol=1e-5)
    # the state of another type, resets as floats, lengths as int32 and beyond the ends
    rs = (torch.rand(40, 3, device=DEV, generator=gen(5)) < 0.2)
    ln = torch.tensor([-5, 7, 1000], device=DEV, dtype=torch.int32)
    h1, hn1 = ops.gated_scan(x, gate, h0.bfloat16(), reset=rs.float(), lengths=ln)
    want = scan64(x, gate, h0.bfloat16(), rs, ln)
    scan_close({"h": h1, "hn": hn1}, want, 40)
    assert torch.equal(hn1[0], h0.bfloat16()[0].float())
    h0b = h0.bfloat16().requires_grad_(True)
    _, hn = ops.gated_scan(x, gate, h0b)
    hn.sum().backward()
    assert h0b.grad.dtype == torch.bfloat16 and h0b.grad.shape == h0.shape


@pytest.mark.parametrize("shape", [(0, 2, 3), (4, 0, 3), (4, 2, 0)], ids=str)
def test_gated_scan_of_nothing(shape):
    T, B, D = shape
    x, gate = (torch.randn(shape, device=DEV, requires_grad=True) for _ in range(2))
    h0 = torch.randn(B, D, device=DEV, requires_grad=True)
    h, hn = ops.gated_scan(x, gate, h0)
    assert h.shape == shape and torch.equal(hn, h0)
    (h.sum() + hn.sum()).backward()
    assert torch.equal(h0.grad, torch.ones_like(h0))


def test_gated_scan_ignores_what_is_masked():
    T, B, D = 150, 3, 66
    x, gate, h0, dh, dhn, _, _ = scan_data(T, B, D, torch.float32, 6)
    ln = torch.tensor([150, 70, 0], device=DEV)
    dead = (torch.arange(T, device=DEV)[:, None] >= ln).unsqueeze(-1).expand(T, B, D)
    want = scan64(x, gate, h0, None, ln, dh, dhn)
    for bad in (float("nan"), float("inf"), torch.finfo(torch.float32).min):
        xb, gb, db = (t.masked_fill(dead, bad) for t in (x, gate, dh))
        got = scan_grads(xb, gb, h0, db, dhn, None, ln)
        scan_close(got, want, T)
        assert bool((got["h"][dead] == 0).all()) and bool((got["dx"][dead] == 0).all())
    # a state that is not finite ends at the next reset, in both directions
    rs = torch.zeros(T, B, dtype=torch.bool, device=DEV)
    rs[100] = True
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[60] = bad
        got = scan_grads(xb, gate, h0, dh, dhn, rs, None)
        want = scan64(x, gate, h0, rs, None, dh, dhn)
        assert not bool(torch.isfinite(got["h"][99]).any())
        scan_close({k: got[k][100:] for k in ("h", "dx", "dgate")} | {"hn": got["hn"], "dh0": got["dh0"]},
                   {k: want[k][100:] for k in ("h", "dx", "dgate")} | {"hn": want["hn"], "dh0": want["dh0"]}, T)
        scan_close({"dx": got["dx"][:60], "dh0": got["dh0"]}, {"dx": want["dx"][:60], "dh0": want["dh0"]}, T)
        db = dh.clone()
        db[120] = bad                # a bad gradient behind the reset stays behind it
        got = scan_grads(x, gate, h0, db, dhn, rs, None)
        scan_close({k: got[k][:100] for k in ("dx", "dgate")} | {"dh0": got["dh0"]},
                   {k: want[k][:100] for k in ("dx", "dgate")} | {"dh0": want["dh0"]}, T)


def test_gated_scan_extreme_gates():
    x, gate, h0, dh, dhn, _, _ = scan_data(30, 2, 64, torch.float32, 7)
    gate[3], gate[7], gate[11], gate[13] = 200., -200., float("inf"), -float("inf")
    got = scan_grads(x, gate, h0, dh, dhn, None, None)
    want = scan64(x, gate, h0, None, None, dh, dhn)
    scan_close(got, want, 404)
    assert torch.equal(got["h"][3], x[3]) and torch.equal(got["h"][11], x[11])
    assert torch.equal(got["h"][7], got["h"][6]) and torch.equal(got["h"][13], got["h"][12])


def test_gated_scan_gradient_against_differences():
    x, gate, h0, dh, dhn, rs, ln = scan_data(50, 2, 40, torch.float32, 8, True, True)
    got = scan_grads(x, gate, h0, dh, dhn, rs, ln)

    def value(x, gate, h0):
        h, hn = ops.gated_scan(x, gate, h0, reset=rs, lengths=ln)
        return float((h.double() * dh).sum() + (hn.double() * dhn).sum())

    eps = 2. ** -7
    for i, k in enumerate(("dx", "dgate", "dh0")):
        args = [x, gate, h0]
        v = torch.randn(args[i].shape, device=DEV, generator=gen(9))
        args[i] = (x, gate, h0)[i] + eps * v
        up = value(*args)
        args[i] = (x, gate, h0)[i] - eps * v
        slope = (up - value(*args)) / (2 * eps)
        # third derivatives of sigmoid chains times eps^2 / 6, and 2^-24 of the sums over 2 eps
        scale = float((got[k].double().abs() * v.abs()).sum())
        assert abs(slope - float((got[k].double() * v).sum())) <= 2e-4 * scale, k


def test_gated_scan_offsets_past_32_bits():
    T, B, D = (1 << 21) + 5, 1, 1056           # 2.2e9 elements a stream
    g = gen(10)
    x = torch.empty(T, B, D, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    gate = torch.empty_like(x).normal_(generator=g)
    rs = torch.zeros(T, B, dtype=torch.bool, device=DEV)
    rs[T - 40] = True
    with torch.no_grad():
        h, hn = ops.gated_scan(x, gate, reset=rs)
    want = scan64(x[-40:], gate[-40:])
    scan_close({"h": h[-40:], "hn": hn}, want, 40)
    x.requires_grad_(True)
    h, hn = ops.gated_scan(x, gate, reset=rs)
    dh = torch.zeros(1, dtype=torch.bfloat16, device=DEV).expand(T, B, D)
    dx, = torch.autograd.grad((h, hn), (x,), (dh, torch.ones_like(hn)))
    want = scan64(x[-40:], gate[-40:], None, None, None, dh[-40:], torch.ones_like(hn))
    scan_close({"dx": dx[-40:], "dh0": want["dh0"].float()}, {"dx": want["dx"], "dh0": want["dh0"]}, 40)
    assert not bool(dx[:-40].any())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1), (3, 5), (2, 64), (7, 130), (256, 512)], ids=str)
def test_gated_scan_step_is_one_step_of_the_scan(size, dtype):
    B, D = size
    x, gate, h0, _, _, _, _ = scan_data(6, B, D, dtype, 11, layout="halves")
    rs = torch.rand(6, B, device=DEV, generator=gen(12)) < 0.3
    state, ys = h0.clone(), []
    version = state._version
    for t in range(6):
        ys.append(ops.gated_scan_step(x[t], gate[t], state, reset=rs[t]))
    assert state._version > version
    want = scan64(x, gate, h0, rs)
    scan_close({"h": torch.stack(ys), "hn": state}, want, 6)
    with torch.no_grad():
        h, hn = ops.gated_scan(x, gate, h0, reset=rs)
    # the same arithmetic up to the association of a fold
    assert torch.allclose(hn, state, rtol=1e-5, atol=1e-6)


def test_gated_scan_step_refusals_on_the_device():
    x = torch.zeros(2, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.gated_scan_step(x, x, torch.zeros(2, 4))            # state on the host
    with pytest.raises(ValueError):
        ops.gated_scan(x[None], x[None], reset=torch.zeros(1, 2, dtype=torch.bool))
    assert ops.gated_scan_step(x[:0], x[:0], x[:0].clone()).shape == (0, 4)


# ------------------------------------------------------------------------------------- policy loss
def loss64(logits, action, old_logp, adv, ref_logp=None, valid=None, lo=0.2, hi=0.2, c_kl=0., c_ent=0.):
    """By torch's autograd in 64 bits, rows of weight 0 left out."""
    V = logits.shape[-1]
    l64 = logits.detach().double().reshape(-1, V).requires_grad_(True)
    n = l64.shape[0]
    w = torch.ones(n, dtype=torch.float64, device=l64.device) if valid is None else valid.double().reshape(-1)
    on = w != 0
    some = on & (l64 > -math.inf).any(-1)
    total = torch.zeros((), dtype=torch.float64, device=l64.device)
    sums = torch.zeros(4, dtype=torch.float64, device=l64.device)
    if bool(some.any()):
        lp = torch.log_softmax(l64[some], -1)
        logp = lp.gather(-1, action.reshape(-1)[some][:, None]).squeeze(-1)
        ent = -(lp.exp() * lp.masked_fill(lp == -math.inf, 0.)).sum(-1)
        a, ww = adv.double().reshape(-1)[some], w[some]
        r = (logp - old_logp.double().reshape(-1)[some]).exp()
        rc = r.clamp(1 - lo, 1 + hi)
        pi = -torch.minimum(r * a, rc * a)
        kl = torch.zeros_like(pi)
        if ref_logp is not None:
            d = ref_logp.double().reshape(-1)[some] - logp
            kl = d.exp() - d - 1
        sums = torch.stack([(v * ww).sum() for v in (pi, kl, ent, (r != rc).double())]) / w.sum()
        total = sums[0] + c_kl * sums[1] - c_ent * sums[2]
        total.backward()
    grad = torch.zeros_like(l64) if l64.grad is None else l64.grad
    return torch.cat([total.detach().reshape(1), sums.detach()]), grad.reshape(logits.shape)


def loss_data(N, V, dtype, seed, kl=True, valid=True, scale=2.):
    g = gen(seed)
    logits = (torch.randn(N, V, device=DEV, generator=g) * scale).to(dtype)
    action = torch.randint(0, V, (N,), device=DEV, generator=g)
    logp = torch.log_softmax(logits.double(), -1).gather(-1, action[:, None]).squeeze(-1)
    drift = torch.randn(N, device=DEV, generator=g).double() * 0.3
    for edge in (math.log(0.8), math.log(1.3)):       # not within the arithmetic's error of a clip border
        drift = torch.where((drift - edge).abs() < 1e-4, drift + 1e-3, drift)
    old = (logp - drift).float()
    adv = torch.randn(N, device=DEV, generator=g)
    ref = (logp + torch.randn(N, device=DEV, generator=g) * 0.3).float() if kl else None
    w = None
    if valid:
        w = (torch.rand(N, device=DEV, generator=g) < 0.7).float() * (0.5 + torch.rand(N, device=DEV, generator=g))
    return logits, action, old, adv, ref, w


def run_loss(logits, action, old, adv, ref, w, **kw):
    logits = logits.detach().requires_grad_(True)
    loss, scalars = ops.policy_kl_loss(logits, action, old, adv, ref_logp=ref, valid=w, **kw)
    loss.backward()
    return loss.detach(), scalars, logits.grad


def loss_close(loss, scalars, grad, want_s, want_g, cancel=0.):
    # a row: |x - max| < 64 in e^(x - max) and 2^-20 for the sum, of terms of the size of the row's largest.  cancel: what
    # the entropy's part c_H p (log p + H) w / sum w consists of: log p and H are each known to err relative, and in a row that
    # is all but uniform and has no other part (a clipped ratio, a tiny advantage) they cancel, the row's largest with them
    err = (64 + 4) * 2. ** -24 + 2. ** -20
    top = want_g.abs().amax(-1, keepdim=True) + cancel
    assert bool(((grad.double() - want_g).abs() <=
                 HALF[grad.dtype] * want_g.abs() + 4 * err * top + torch.finfo(grad.dtype).tiny).all()), \
        float(((grad.double() - want_g).abs() - HALF[grad.dtype] * want_g.abs()).max())
    size = want_s.abs().max() + 1
    assert bool(((scalars.double() - want_s).abs() <= (err + 2. ** -23) * 4 * size).all()), (scalars, want_s)
    assert torch.equal(loss, scalars[0])


KW = dict(clip_low=0.2, clip_high=0.3)
LOSS_SIZES = [(1, 1), (1, 2), (5, 3), (700, 6), (33, 8), (1000, 18), (37, 33), (9, 64), (70, 65), (19, 129), (7, 255),
              (40, 256), (6, 1000), (3, 1024), (3, 1025), (130, 1500), (200, 4099), (130, 9001), (140, 20000),
              (129, 40000), (2, 32771), (128, 70001), (128, 100003), (1, 131072), (3, 300007)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", LOSS_SIZES, ids=str)
def test_policy_kl_loss(size, dtype):
    N, V = size
    kl, valid = (N + V) % 3 != 0, (N + V) % 2 == 0
    data = loss_data(N, V, dtype, 20 + N, kl, valid)
    c = dict(kl_coeff=0.1 if kl else 0., entropy_coeff=0.02)
    out = run_loss(*data, **KW, **c)
    logits, action, old, adv, ref, w = data
    want = loss64(logits, action, old, adv, ref, w, 0.2, 0.3, c["kl_coeff"], 0.02)
    loss_close(*out, *want)
    # without a gradient: the same numbers
    with torch.no_grad():
        loss, scalars = ops.policy_kl_loss(logits, action, old, adv, ref_logp=ref, valid=w, **KW, **c)
    assert torch.equal(scalars, out[1])
    lp, ent = ops.action_logp(logits, action)
    l64 = torch.log_softmax(logits.double(), -1)
    want_lp = l64.gather(-1, action[:, None]).squeeze(-1)
    tol = 2. ** -20 + 68 * 2. ** -24
    assert bool(((lp.double() - want_lp).abs() <= tol + want_lp.abs() * 2. ** -24).all())
    want_ent = -(l64.exp() * l64).sum(-1)
    assert bool(((ent.double() - want_ent).abs() <= tol * (1 + want_ent)).all())


@pytest.mark.parametrize("size", [(4, 2, 18), (4, 3, 2000), (3, 5, 20000)], ids=str)
def test_policy_kl_loss_shapes_strides_and_types(size):
    T, B, V = size
    g = gen(30)
    wide = torch.randn(T, B, V + 5, device=DEV, generator=g)
    logits = wide[..., 2:V + 2]                            # rows farther apart than V, odd starts
    flat = logits.reshape(-1, V)
    _, action, old, adv, ref, w = loss_data(T * B, V, torch.float32, 31)
    action = torch.randint(0, V, (T, B), device=DEV, generator=g, dtype=torch.int32)
    old, adv, ref, w = (t.reshape(T, B) for t in (old, adv, ref, w))
    mask = w > 0.8
    want = loss64(flat, action.long(), old, adv, ref, mask, 0.2, 0.3, 0.1, 0.01)
    leaf = logits.detach()
    leaf.requires_grad_(True)
    loss, scalars = ops.policy_kl_loss(leaf, action, old.double(), adv, ref_logp=ref, valid=mask, kl_coeff=0.1,
                                       entropy_coeff=0.01, **KW)
    loss.backward()
    loss_close(loss.detach(), scalars, leaf.grad.reshape(-1, V), want[0], want[1].reshape(-1, V))
    # logits without a unit stride along V, and rows that are one and the same
    turned = flat.t().contiguous().t()
    out = run_loss(turned, action.reshape(-1), old.reshape(-1), adv.reshape(-1), ref.reshape(-1), mask.reshape(-1),
                   kl_coeff=0.1, entropy_coeff=0.01, **KW)
    assert torch.equal(out[1], scalars)
    same = flat[:1].expand(6, V)
    lp, _ = ops.action_logp(same, torch.zeros(6, dtype=torch.long, device=DEV))
    assert bool((lp == lp[0]).all())


@pytest.mark.parametrize("V", [7, 18, 500, 3000, 140000])
def test_policy_kl_loss_masked_rows_and_actions(V):
    N = 12
    logits, action, old, adv, ref, _ = loss_data(N, V, torch.float32, 40)
    ban = torch.rand(N, V, device=DEV, generator=gen(41)) < 0.4
    ban.scatter_(-1, action[:, None], False)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        masked = logits.masked_fill(ban, low)
        w = torch.ones(N, device=DEV)
        w[3] = w[7] = 0
        args = dict(kl_coeff=0.1, entropy_coeff=0.02)
        want = loss64(logits.masked_fill(ban, -1e30), action, old, adv, ref, w, 0.2, 0.3, 0.1, 0.02)
        out = run_loss(masked, action, old, adv, ref, w, **KW, **args)
        loss_close(*out, *want)
        assert not bool(out[2][ban].any())
        # what stands in rows without weight is not read: NaN, infinities, actions out of range
        bad, bad_a, bad_old = masked.clone(), action.clone(), old.clone()
        bad[3], bad[7] = float("nan"), float("inf")
        bad_a[3], bad_a[7], bad_old[3] = -100, V + 5, float("nan")
        again = run_loss(bad, bad_a, bad_old, adv, ref, w, **KW, **args)
        assert torch.equal(again[1], out[1]) and torch.equal(again[2], out[2])
    # nothing valid
    loss, scalars, grad = run_loss(logits, action, old, adv, ref, torch.zeros(N, device=DEV), **KW)
    assert not bool(scalars.any()) and not bool(grad.any()) and float(loss) == 0.
    # a row that allows nothing adds nothing, and counts in the mean
    none = logits.clone()
    none[5] = -math.inf
    want = loss64(none, action, old, adv, ref, None, 0.2, 0.3, 0.1, 0.02)
    out = run_loss(none, action, old, adv, ref, None, kl_coeff=0.1, entropy_coeff=0.02, **KW)
    loss_close(*out, *want)
    assert not bool(out[2][5].any())
    lp, ent = ops.action_logp(none, action)
    assert float(lp[5]) == -math.inf and float(ent[5]) == 0.
    # a valid row with an action out of range, or a NaN: loud
    for spoil in ("action", "logit"):
        l2, a2 = logits.clone(), action.clone()
        if spoil == "action":
            a2[2] = V
        else:
            l2[2, V // 2] = float("nan")
        loss, _, _ = run_loss(l2, a2, old, adv, ref, None, **KW)
        assert math.isnan(float(loss))
    lp, _ = ops.action_logp(logits, torch.full_like(action, -1))
    assert bool(torch.isnan(lp).all())


def test_policy_kl_loss_far_logits_and_ratios():
    N, V = 64, 50
    logits, action, old, adv, ref, _ = loss_data(N, V, torch.float32, 50, scale=30.)
    out = run_loss(logits + 1000., action, old, adv, ref, None, entropy_coeff=0.02, kl_coeff=0.1, **KW)
    shifted = (logits + 1000.)
    want = loss64(shifted, action, old, adv, ref, None, 0.2, 0.3, 0.1, 0.02)
    # log-probabilities down to -200 here: kl of d = ref - logp is known to e^d |delta d|
    assert torch.allclose(out[1].double(), want[0], rtol=1e-3)
    # a ratio that overflows: the clipped branch wins for positive advantages, advantage 0 adds nothing
    old = torch.full((N,), -3e38, device=DEV)
    adv = torch.where(torch.arange(N, device=DEV) % 2 == 0, 1., 0.)
    loss, scalars, grad = run_loss(logits, action, old, adv, None, None, **KW)
    assert abs(float(loss) + 1.3 * 0.5) < 1e-6 and not bool(grad.any())


def test_policy_kl_loss_sums_over_many_rows(N=20000, V=200, dtype=torch.float32):
    # more rows than one workgroup adds: shares first.  (Sums over rows are 64 bits, so the tolerances do not grow.)
    data = loss_data(N, V, dtype, 52)
    c = dict(kl_coeff=0.1, entropy_coeff=0.02)
    logits, action, old, adv, ref, w = data
    # a row's gradient is w / sum w times p or 1 - p times the sum of -r A, -0.1 (e^d - 1) and 0.02 (log p + H): with log p known
    # to err, r and e^d are to err relative; in some of many rows the three cancel to less than err of their sizes
    lp = torch.log_softmax(logits.double(), -1).gather(-1, action[:, None]).squeeze(-1)
    parts = (lp - old).exp() * adv.abs() + 0.1 * ((ref - lp).exp() + 1.) + 0.02 * math.log(V)
    loss_close(*run_loss(*data, **KW, **c), *loss64(*data, 0.2, 0.3, 0.1, 0.02),
               cancel=(parts * w / w.double().sum())[:, None])


def test_policy_kl_loss_weights_summed_in_a_launch_of_their_own():
    test_policy_kl_loss_sums_over_many_rows(4000, 200)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [5, 30, 100, 900, 3500, 40000])
def test_policy_kl_loss_of_huge_logits(V, dtype):
    """Masks of the type's lowest value and others, also over whole rows, are logits like all others: a row of equal ones is
    uniform.  2^20 ln 2 = 726817 is where another expression takes over."""
    N, least, most = 10, torch.finfo(dtype).min, torch.finfo(dtype).max
    noise = torch.randn(N, V, device=DEV, generator=gen(55)).double()
    logits = torch.zeros(N, V, device=DEV, dtype=torch.float64)
    logits[0], logits[1], logits[2], logits[3] = least, -1e30, most, 1e30
    logits[4] = least
    logits[4, V // 2] = 0.5
    logits[5] = -1e9 + 100. * noise[5]
    logits[6], logits[7] = 726817. + noise[6], -726817. + noise[7]
    logits[8] = least
    logits[8, ::2] = -math.inf
    logits[9] = noise[9]
    logits[9, 1::2] = least
    logits = logits.clamp(least, most).masked_fill(logits == -math.inf, -math.inf).to(dtype)
    action = logits.argmax(-1)
    l64 = torch.log_softmax(logits.double(), -1)
    want = l64.gather(-1, action[:, None]).squeeze(-1)
    lp, ent = ops.action_logp(logits, action)
    tol = 2. ** -20 + 68 * 2. ** -24               # as in test_policy_kl_loss
    assert bool(((lp.double() - want).abs() <= tol + want.abs() * 2. ** -24).all()), (lp, want)
    want_ent = -(l64.exp() * l64.clamp(min=-1e300)).sum(-1)
    assert bool(((ent.double() - want_ent).abs() <= tol * (1 + want_ent)).all()), (ent, want_ent)
    g = gen(56)
    old, ref = (want + 0.1 * torch.rand(N, device=DEV, generator=g)).float(), (want + 0.2).float()
    adv = torch.randn(N, device=DEV, generator=g)
    out = run_loss(logits, action, old, adv, ref, None, kl_coeff=0.1, **KW)
    loss_close(*out, *loss64(logits, action, old, adv, ref, None, 0.2, 0.3, 0.1))


def test_policy_kl_loss_gradient_against_differences():
    logits, action, old, adv, ref, w = loss_data(40, 300, torch.float32, 60)
    c = dict(kl_coeff=0.3, entropy_coeff=0.2)
    _, _, grad = run_loss(logits, action, old, adv, ref, w, **KW, **c)
    v = torch.randn(40, 300, device=DEV, generator=gen(61))
    eps = 2. ** -8

    def value(s):
        return float(ops.policy_kl_loss(logits + s * eps * v, action, old, adv, ref_logp=ref, valid=w, **KW, **c)[0])

    slope = (value(1) - value(-1)) / (2 * eps)
    # 2^-24 of a loss of order 1 over 2 eps, the curvature, and the rows whose ratio crosses a clip border on the way
    scale = float((grad.double().abs() * v.abs()).sum())
    assert abs(slope - float((grad.double() * v).sum())) <= 2e-2 * scale


def test_policy_kl_loss_backward_scale_and_second_pass():
    data = loss_data(20, 900, torch.float32, 70)
    _, _, grad = run_loss(*data, **KW)
    logits = data[0].clone().requires_grad_(True)
    call = lambda: ops.policy_kl_loss(logits, *data[1:4], ref_logp=data[4], valid=data[5], **KW)[0]  # noqa: E731
    (call() * 0.25).backward()
    assert torch.equal(logits.grad, grad * 0.25)
    logits.grad = None
    one = ops.unit_seed(logits.device)
    torch.autograd.backward(call(), one)
    assert torch.equal(logits.grad, grad)
    logits.grad = None
    loss = ops.policy_kl_loss(logits, *data[1:4], ref_logp=data[4], valid=data[5], grad_scale=1024., **KW)[0]
    (1024. * loss).backward()
    assert torch.equal(logits.grad, grad * 1024.)
    logits.grad = None
    ops.policy_kl_loss(logits, *data[1:4], ref_logp=data[4], valid=data[5], grad_scale=1024., **KW)[0].backward()
    assert torch.equal(logits.grad, grad)
    loss = call()
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="first backward"):
        loss.backward()
    # nothing at all
    empty = torch.zeros(0, 5, device=DEV, requires_grad=True)
    none = torch.zeros(0, device=DEV)
    loss, scalars = ops.policy_kl_loss(empty, none.long(), none, none)
    loss.backward()
    assert float(loss.detach()) == 0. and empty.grad.shape == (0, 5)


def test_policy_kl_loss_float16_gradients_that_underflow_unscaled():
    N, V, S = 2000, 3000, 65536.
    logits, action, old, adv, ref, _ = loss_data(N, V, torch.float16, 71)
    leaf = logits.clone().requires_grad_(True)
    loss, _ = ops.policy_kl_loss(leaf, action, old, adv, ref_logp=ref, grad_scale=S, **KW)
    (loss * S).backward()
    _, want = loss64(logits, action, old, adv, ref, None, 0.2, 0.3)
    want = want * S
    err = (64 + 4) * 2. ** -24 + 2. ** -20          # as in loss_close, beside float16's subnormals: steps of 2^-24
    assert bool(((leaf.grad.double() - want).abs() <= HALF[torch.float16] * want.abs() + 2. ** -25
                 + 4 * err * want.abs().amax(-1, keepdim=True)).all())
    assert bool((leaf.grad != 0)[want.abs() > 2. ** -24].all())          # nothing that float16 holds is lost


def test_policy_kl_loss_many_rows_go_in_slices():
    N, V = (1 << 21) + 70, 3
    g = gen(72)
    logits = torch.randn(N, V, device=DEV, generator=g)
    action = torch.randint(0, V, (N,), device=DEV, generator=g)
    old = torch.log_softmax(logits, -1).gather(-1, action[:, None]).squeeze(-1) - 0.05
    adv = torch.randn(N, device=DEV, generator=g)
    out = run_loss(logits, action, old, adv, None, None, entropy_coeff=0.02, **KW)
    want = loss64(logits, action, old, adv, None, None, 0.2, 0.3, 0., 0.02)
    loss_close(*out, *want, cancel=0.02 * math.log(3) / N)


def test_policy_kl_loss_of_one_row_without_leading_axes():
    logits = torch.randn(50, device=DEV, generator=gen(73), requires_grad=True)
    action = torch.tensor(7, device=DEV)
    old, ent = ops.action_logp(logits.detach(), action)
    assert old.shape == () and ent.shape == ()
    loss, _ = ops.policy_kl_loss(logits, action, old, torch.tensor(2., device=DEV))
    loss.backward()
    assert logits.grad.shape == (50,) and abs(float(loss.detach()) + 2.) < 1e-5


def test_second_derivatives_are_refused():
    x = torch.randn(5, 2, 4, device=DEV, requires_grad=True)
    gate = torch.randn(5, 2, 4, device=DEV)
    h, _ = ops.gated_scan(x, gate)
    g, = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    want, = torch.autograd.grad(ops.gated_scan(x, gate)[0].sum(), x)
    assert torch.equal(g.detach(), want)


def test_policy_kl_loss_offsets_past_32_bits():
    N, V = 35000, 65536                                  # 2.3e9 logits
    g = gen(80)
    logits = torch.empty(N, V, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    action = torch.randint(0, V, (N,), device=DEV, generator=g)
    old, adv = torch.full((N,), -11., device=DEV), torch.ones(N, device=DEV)
    w = torch.zeros(N, device=DEV)
    w[-3:] = 1.
    logits.requires_grad_(True)
    loss, scalars = ops.policy_kl_loss(logits, action, old, adv, valid=w, **KW)
    grad, = torch.autograd.grad(loss, logits)
    want = loss64(logits[-3:], action[-3:], old[-3:], adv[-3:], None, None, 0.2, 0.3)
    loss_close(loss.detach(), scalars, grad[-3:], *want)
    assert not bool(grad[-4].any()) and not bool(grad[0].any())


# ------------------------------------------------------------------------------------- orthogonalize
def orth64(g, steps=5, coeffs=ops.orthogonalize.__defaults__[1], eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


def orth_close(got, want):
    m = min(got.shape)
    norm = float(want.norm())
    # pieces of 22 bits: 2^-23 of |X| = 1, times 484, in a result of norm ~ sqrt(m); some of the rounding doubles it
    err = 4 * 484 * 2. ** -23 / max(1., math.sqrt(m))
    off = (got.double() - want - 0.)
    allowed = HALF[got.dtype] * norm + err * norm
    assert float(off.norm()) <= allowed, (float(off.norm()) / norm, err)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1), (1, 50), (3, 2), (16, 256), (64, 576), (127, 129), (128, 128), (129, 127), (512, 18),
                                  (300, 1000), (1000, 130), (700, 700)], ids=str)
def test_orthogonalize(size, dtype):
    g = torch.randn(*size, device=DEV, generator=gen(90)).to(dtype) * 0.01
    got = ops.orthogonalize(g)
    assert got.shape == g.shape and got.dtype == dtype and got.is_contiguous()
    orth_close(got, orth64(g))


def test_orthogonalize_of_lists_batches_and_views():
    mk = gen(91)
    mats = [torch.randn(*s, device=DEV, generator=mk) for s in ((5, 9), (3, 40, 70), (2, 2, 130, 20), (0, 4), (256, 100))]
    mats.append(torch.randn(50, 60, device=DEV, generator=mk).bfloat16())
    mats.append(torch.randn(90, 64, device=DEV, generator=mk).t())            # transposed
    mats.append(torch.randn(90, 64, device=DEV, generator=mk)[5:50, 3:40])    # rows farther apart
    mats += [torch.randn(10 + k, 33, device=DEV, generator=mk) for k in range(40)]    # more than one table
    mats.append(mats[0])                                                      # the same one twice
    outs = ops.orthogonalize(mats)
    assert len(outs) == len(mats)
    for g, o in zip(mats, outs):
        assert o.shape == g.shape and o.dtype == g.dtype
        if g.numel() == 0:
            continue
        for gi, oi in zip(g.reshape(-1, *g.shape[-2:]), o.reshape(-1, *g.shape[-2:])):
            orth_close(oi, orth64(gi))
    assert torch.equal(outs[0], outs[-1])
    alone = ops.orthogonalize(mats[1])
    assert torch.equal(alone, outs[1])       # (these few are too small to be split differently in company)


def test_orthogonalize_options_and_edges():
    g = torch.randn(40, 80, device=DEV, generator=gen(92))
    for steps, coeffs in ((1, (1.5, -0.5, 0.)), (12, (1.5, -0.5, 0.)), (3, (2., -1.5, 0.5))):
        orth_close(ops.orthogonalize(g, steps=steps, coeffs=coeffs), orth64(g, steps, coeffs))
    assert not bool(ops.orthogonalize(torch.zeros(30, 20, device=DEV)).any())
    for size in (1e-3, 1e3, 1e18):           # the norm goes out before anything is rounded
        orth_close(ops.orthogonalize(g * size, eps=0.), orth64(g, eps=0.))
    bad = g.clone()
    bad[3, 4] = float("nan")
    assert bool(torch.isnan(ops.orthogonalize(bad)).any())
    for size in (1e-36, 1e36):               # a reciprocal norm beyond 32 bits
        orth_close(ops.orthogonalize(g * size, eps=0.), orth64(g * size, eps=0.))
    assert not bool(ops.orthogonalize(torch.zeros(30, 20, device=DEV), eps=0.).any())
    low = g[:, :1] @ g[:1, :]                # rank 1: the noise of the products is amplified 484 times
    got, want = ops.orthogonalize(low), orth64(low)
    assert float((got.double() - want).norm()) <= 484 * 2. ** -22 * 4 * float(want.norm())
    with pytest.raises(_lib.HipError, match="range of the stored factors"):
        ops.orthogonalize(g, coeffs=(9., 0., 0.))


def test_orthogonalize_large_has_singular_values_near_one():
    g = torch.randn(1500, 2100, device=DEV, generator=gen(93))
    got = ops.orthogonalize(g)
    orth_close(got, orth64(g))
    s = torch.linalg.svdvals(got.double().cpu()[:, :])
    assert 0.3 < float(s.min()) and float(s.max()) < 1.3


# ------------------------------------------------------------------------------------- together, streams and graphs
def test_operators_replayed_in_a_graph_while_eager_work_runs():
    x, gate, h0, dh, dhn, rs, ln = scan_data(300, 2, 64, torch.float32, 100, True, True)
    logits, action, old, adv, ref, w = loss_data(30, 3000, torch.float32, 101)
    mats = [torch.randn(70, 90, device=DEV, generator=gen(102)), torch.randn(30, 10, device=DEV, generator=gen(103))]
    xs, gs, hs, ls = (t.clone().requires_grad_(True) for t in (x, gate, h0, logits))
    ms = [m.clone() for m in mats]
    state = h0.clone()

    def work():
        h, hn = ops.gated_scan(xs, gs, hs, reset=rs, lengths=ln)
        grads = torch.autograd.grad((h, hn), (xs, gs, hs), (dh, dhn))
        loss, scalars = ops.policy_kl_loss(ls, action, old, adv, ref_logp=ref, valid=w, kl_coeff=0.1, entropy_coeff=0.01)
        g, = torch.autograd.grad(loss, ls)
        y = ops.gated_scan_step(x[0], gate[0], state)
        return [t.detach() for t in (h, hn, *grads, scalars, g, *ops.orthogonalize(ms), y)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for k in range(4):
        with torch.no_grad():
            for dst, src in ((xs, x), (gs, gate), (ls, logits), (ms[0], mats[0])):
                dst.copy_(src * (1 + k) / 2)
            state.copy_(h0)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        state.copy_(h0)
        want = work()                       # eager work of the same operators between the replays
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_backward_pass_captured_with_its_leaves():
    """``loss.backward()`` into ``.grad`` within a graph: a projection, the scan, the loss."""
    T, B, D, V = 40, 3, 32, 50
    g = gen(105)
    feed = torch.randn(T, B, D, device=DEV, generator=g)
    w = (torch.randn(2 * D, D, device=DEV, generator=g) * 0.2).requires_grad_(True)
    head = (torch.randn(V, D, device=DEV, generator=g) * 0.2).requires_grad_(True)
    action = torch.randint(0, V, (T, B), device=DEV, generator=g)
    old, adv = torch.full((T, B), -4., device=DEV), torch.randn(T, B, device=DEV, generator=g)

    def work(w, head):
        x, gate = torch.nn.functional.linear(feed, w).chunk(2, -1)
        h, _ = ops.gated_scan(x, gate)
        loss, scalars = ops.policy_kl_loss(torch.nn.functional.linear(h, head), action, old, adv, entropy_coeff=0.01)
        loss.backward()
        return scalars

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work(w, head)
    torch.cuda.current_stream().wait_stream(side)
    w.grad = head.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scalars = work(w, head)
    for k in range(4):
        feed.mul_(1. + 0.1 * k)
        graph.replay()
        torch.cuda.synchronize()
        other = [t.detach().clone().requires_grad_(True) for t in (w, head)]
        want = work(*other)
        assert torch.equal(scalars, want)
        # (the library's products of an eager call may be other kernels than the captured ones': 2^-24 of up to 120 terms)
        for a, b in zip((w, head), other):
            assert torch.allclose(a.grad, b.grad, rtol=1e-4, atol=1e-6)


def test_capture_is_refused_while_an_eager_graph_of_the_leaf_lives():
    x, gate = (torch.randn(4, 2, 8, device=DEV, generator=gen(106)).requires_grad_(True) for _ in range(2))
    logits = torch.randn(4, 9, device=DEV, generator=gen(107)).requires_grad_(True)
    action, zero = torch.zeros(4, dtype=torch.long, device=DEV), torch.zeros(4, device=DEV)
    calls = (lambda: ops.gated_scan(x, gate), lambda: ops.policy_kl_loss(logits, action, zero, zero))
    for call in calls:
        held = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="drop it before"):
            with torch.cuda.graph(graph):
                call()
        with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):    # without a backward pass it may be captured
            call()
        del held
        call()                               # and eager calls go on


def test_operators_on_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    datas = [scan_data(3000, 1, 130, torch.bfloat16, 110 + k, True) for k in range(2)]
    losses = [loss_data(20, 60000, torch.float32, 112 + k) for k in range(2)]
    mats = [torch.randn(200, 300, device=DEV, generator=gen(114 + k)) for k in range(2)]
    want = [(scan_grads(*d), run_loss(*q, **KW), ops.orthogonalize(m)) for d, q, m in zip(datas, losses, mats)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, d, q, m in zip(streams, datas, losses, mats):
            with torch.cuda.stream(s):
                got.append((scan_grads(*d), run_loss(*q, **KW), ops.orthogonalize(m)))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(g[0][k], w[0][k]) for k in w[0])
            assert all(torch.equal(a, b) for a, b in zip(g[1], w[1])) and torch.equal(g[2], w[2])


def test_results_do_not_depend_on_the_run():
    d = scan_data(2000, 2, 200, torch.float16, 120, True, True)
    q = loss_data(300, 5000, torch.bfloat16, 121)
    first = (scan_grads(*d), run_loss(*q, **KW))
    for _ in range(2):
        again = (scan_grads(*d), run_loss(*q, **KW))
        assert all(torch.equal(again[0][k], first[0][k]) for k in first[0])
        assert all(torch.equal(a, b) for a, b in zip(again[1], first[1]))


# ------------------------------------------------------------------------------------- Muon, and all of it together
def muon64(p, grads, lr, beta, nesterov, decay):
    p, buf = p.double(), torch.zeros_like(p, dtype=torch.float64)
    for g in grads:
        g = g.double()
        buf = beta * buf + (1 - beta) * g
        u = g + beta * (buf - g) if nesterov else buf
        o = orth64(u.reshape(u.shape[0], -1)).reshape(p.shape)
        m, n = p.shape[0], p[0].numel()
        p = p * (1 - lr * decay) - lr * math.sqrt(max(1., m / n)) * o
    return p


@pytest.mark.parametrize("nesterov,decay", [(True, 0.), (False, 0.1)])
def test_muon_steps(nesterov, decay):
    from rlpyt_amd.optim import Muon
    mk = gen(130)
    shapes = [(40, 70), (96, 30), (16, 4, 8, 8), (12,), (1, 5)]
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV, generator=mk)) for s in shapes]
    start = [p.detach().clone() for p in params]
    grads = [[torch.randn(*s, device=DEV, generator=mk) for s in shapes] for _ in range(3)]
    opt = Muon(params, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    for gs in grads:
        for p, g in zip(params, gs):
            p.grad = g.clone()
        norm = opt.clip_and_step(None)
        want = torch.sqrt(sum(g.double().square().sum() for g in gs))
        assert abs(float(norm) / float(want) - 1) < 1e-5
    for k, (p, s) in enumerate(zip(params, start)):
        if p.dim() < 2:
            continue
        want = muon64(s, [gs[k] for gs in grads], 0.02, 0.9, nesterov, decay)
        # three updates of lr x (a matrix' tolerance), and 2^-24 of the weights each
        err = 3 * 0.02 * 4 * 484 * 2. ** -23 * math.sqrt(max(1., p.shape[0] / p[0].numel())) + 6 * 2. ** -24 * float(want.norm())
        assert float((p.detach().double() - want).norm()) <= err
    # vectors: Adam's first step is lr_adam * sign(g)
    q = torch.nn.Parameter(torch.zeros(7, device=DEV))
    q.grad = torch.randn(7, device=DEV, generator=mk)
    Muon([q], lr=0.02, adam_lr_ratio=0.05).step()
    assert torch.allclose(q.detach(), -0.001 * q.grad.sign(), rtol=1e-4)
    # a state dict carries on
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt2 = Muon(other, lr=0.5)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, o, g in zip(params, other, grads[0]):
        p.grad, o.grad = g.clone(), g.clone()
    opt.clip_and_step(1.)
    opt2.clip_and_step(1.)
    assert all(torch.equal(p, o) for p, o in zip(params, other))


def test_muon_of_16_bit_parameters_keeps_its_buffers_in_32():
    from rlpyt_amd.optim import Muon
    mk = gen(131)
    w = torch.nn.Parameter(torch.randn(60, 90, device=DEV, generator=mk).bfloat16())
    v = torch.nn.Parameter(torch.zeros(9, device=DEV, dtype=torch.bfloat16))
    start = w.detach().clone()
    opt = Muon([w, v], lr=0.5)
    grads = [torch.randn(60, 90, device=DEV, generator=mk).bfloat16() for _ in range(2)]
    for g in grads:
        w.grad, v.grad = g.clone(), torch.ones_like(v)
        opt.step()
    assert opt.state[w]["momentum_buffer"].dtype == torch.float32 == opt.state[v]["exp_avg"].dtype
    want = muon64(start, grads, 0.5, 0.95, True, 0.)
    # two roundings of the weights, beside the updates' own error
    err = 2 * HALF[torch.bfloat16] * float(want.norm()) + 2 * 0.5 * 4 * 484 * 2. ** -23
    assert float((w.detach().double() - want).norm()) <= err
    other = Muon([torch.nn.Parameter(w.detach().clone()), torch.nn.Parameter(v.detach().clone())])
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    buf = other.state[other.param_groups[0]["params"][0]]["momentum_buffer"]
    assert buf.dtype == torch.float32 and torch.equal(buf, opt.state[w]["momentum_buffer"])


def test_muon_of_empty_and_missing_gradients():
    from rlpyt_amd.optim import Muon
    ps = [torch.zeros(3, 0, device=DEV, requires_grad=True), torch.ones(4, 5, device=DEV, requires_grad=True),
          torch.ones(6, 2, device=DEV, requires_grad=True), torch.zeros(0, device=DEV, requires_grad=True)]
    opt = Muon(ps)
    opt.step()                               # no gradient at all
    for p in (ps[0], ps[1], ps[3]):
        p.grad = torch.ones_like(p)
    norm = opt.clip_and_step(1.)
    assert abs(float(norm) - math.sqrt(20)) < 1e-5
    assert bool((ps[1] < 1).all()) and bool((ps[2] == 1).all()) and ps[0].shape == (3, 0)


def test_a_recurrent_policy_trains_with_the_operators_together():
    """Embedding, gated recurrence over time with resets and padding, logits, loss, Muon: gradients of every
    parameter against the same network in 64 bits, an update, and the sampler's one-step form on the way."""
    from rlpyt_amd.optim import Muon
    T, B, I, D, V = 60, 5, 24, 96, 200
    mk = gen(140)
    w_in = torch.nn.Parameter(torch.randn(2 * D, I, device=DEV, generator=mk) / I ** 0.5)
    bias = torch.nn.Parameter(torch.randn(2 * D, device=DEV, generator=mk) * 0.1)
    w_out = torch.nn.Parameter(torch.randn(V, D, device=DEV, generator=mk) / D ** 0.5)
    obs = torch.randn(T, B, I, device=DEV, generator=mk)
    reset = torch.rand(T, B, device=DEV, generator=mk) < 0.05
    lengths = torch.tensor([60, 31, 1, 0, 60], device=DEV)
    valid = (torch.arange(T, device=DEV)[:, None] < lengths)
    h0 = torch.randn(B, D, device=DEV, generator=mk)
    adv = torch.randn(T, B, device=DEV, generator=mk)
    with torch.no_grad():            # sampling: one step at a time
        state, steps = h0.clone(), []
        for t in range(T):
            x, gate = torch.nn.functional.linear(obs[t], w_in, bias).chunk(2, -1)
            steps.append(ops.gated_scan_step(x, gate, state, reset=reset[t]))
        logits = torch.nn.functional.linear(torch.stack(steps), w_out)
        action = torch.randint(0, V, (T, B), device=DEV, generator=mk)
        old, _ = ops.action_logp(logits, action)
        old = old + 0.1 * torch.randn(T, B, device=DEV, generator=mk)
    ref = old + 0.1
    x, gate = torch.nn.functional.linear(obs, w_in, bias).chunk(2, -1)
    h, _ = ops.gated_scan(x, gate, h0, reset=reset, lengths=lengths)
    live = valid.unsqueeze(-1)
    assert torch.allclose(torch.where(live, h, torch.zeros_like(h)), torch.where(live, torch.stack(steps), torch.zeros_like(h)),
                          rtol=1e-4, atol=1e-5)
    loss, scalars = ops.policy_kl_loss(torch.nn.functional.linear(h, w_out), action, old, adv, ref_logp=ref,
                                       valid=valid, kl_coeff=0.1, entropy_coeff=0.01)
    loss.backward()
    # the same in 64 bits
    p64 = [p.detach().double().requires_grad_(True) for p in (w_in, bias, w_out)]
    proj = obs.double() @ p64[0].t() + p64[1]
    s, hs = h0.double(), []
    for t in range(T):
        z = torch.sigmoid(proj[t, :, D:])
        k = s * (~reset[t]).unsqueeze(-1)
        new = (1 - z) * k + z * proj[t, :, :D]
        s = torch.where(live[t], new, s)
        hs.append(torch.where(live[t], new, torch.zeros_like(new)))
    lp = torch.log_softmax(torch.stack(hs) @ p64[2].t(), -1)
    logp = lp.gather(-1, action.unsqueeze(-1)).squeeze(-1)
    r = (logp - old.double()).exp()
    d = ref.double() - logp
    each = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (d.exp() - d - 1) + 0.01 * (lp.exp() * lp).sum(-1)
    want = (each * valid).sum() / valid.sum()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    for p, q in zip((w_in, bias, w_out), p64):
        # f32 products of 24 .. 200 terms around the operators
        assert float((p.grad.double() - q.grad).norm()) <= 1e-5 * float(q.grad.norm()), p.shape
    before = w_in.detach().clone()
    opt = Muon([w_in, bias, w_out], lr=0.02)
    opt.clip_and_step(1.0)
    moved = w_in.detach() - before
    assert 0.5 < float(moved.norm()) / (0.02 * math.sqrt(2 * D / I) * math.sqrt(I)) < 1.3


def test_ppo_takes_muon_as_its_optimizer():
    from rlpyt_amd.algos.pg.ppo import PPO
    from rlpyt_amd.optim import Muon
    algo = PPO(OptimCls=Muon, optim_kwargs=dict(momentum=0.9), learning_rate=0.02)
    params = [torch.nn.Parameter(torch.randn(20, 30, device=DEV)), torch.nn.Parameter(torch.zeros(20, device=DEV))]
    algo.optimizer = algo.make_optimizer(params, algo.OptimCls, algo.learning_rate, algo.optim_kwargs)
    assert isinstance(algo.optimizer, Muon) and algo.optimizer.param_groups[0]["momentum"] == 0.9
    for p in params:
        p.grad = torch.randn_like(p)
    out = torch.zeros(1, device=DEV)
    norm = algo.optimizer.clip_and_step(algo.clip_grad_norm, norm_out=out)
    assert float(norm) > 1. and norm is out
    assert float(torch.nn.utils.get_total_norm([p.grad for p in params])) < 1.01 if hasattr(torch.nn.utils, "get_total_norm") else True
    assert isinstance(algo.clip_and_step(), torch.Tensor)


@pytest.mark.parametrize("V", [5, 500, 20000, 40000, 70000])
def test_policy_kl_loss_of_an_empty_batch(V):
    """Rows of every plan: by groups, waves, workgroups and split (past 128 KB and past 256 KB in float32)."""
    logits = torch.zeros(0, V, device=DEV, requires_grad=True)
    none = torch.zeros(0, device=DEV)
    for valid in (None, none):
        loss, scalars = ops.policy_kl_loss(logits, none.long(), none, none, valid=valid, entropy_coeff=0.01)
        grad, = torch.autograd.grad(loss, logits)
        assert float(loss.detach()) == 0. and not bool(scalars.any()) and grad.shape == (0, V)
        with torch.no_grad():
            loss, scalars = ops.policy_kl_loss(logits, none.long(), none, none, valid=valid)
        assert float(loss) == 0. and not bool(scalars.any())
    lp, ent = ops.action_logp(logits.detach(), none.long())
    assert lp.shape == (0,) and ent.shape == (0,)


@pytest.mark.parametrize("layout", ["dense", "batch first", "halves", "odd start"])
def test_gated_scan_results_may_be_written_in_place(layout):
    """As any operator's: the states are a tensor of their own, also where they lie in memory like a [B, T, D] input."""
    x, gate, h0, dh, dhn, rs, ln = scan_data(70, 3, 34, torch.float32, 150, True, True, layout)
    plain = scan_grads(x, gate, h0, dh, dhn, rs, ln)
    leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0)]
    h, hn = ops.gated_scan(*leaves, reset=rs, lengths=ln)
    h.mul_(2.)
    hn.add_(1.)
    assert torch.equal(h.detach(), 2. * plain["h"].detach()) and torch.equal(hn.detach(), plain["hn"].detach() + 1.)
    grads = torch.autograd.grad((h, hn), leaves, (dh, dhn))
    again = torch.autograd.grad(ops.gated_scan(*leaves, reset=rs, lengths=ln), leaves, (2. * dh, dhn))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("V", [7, 18, 100, 500, 3000, 20000, 140000])
def test_policy_kl_loss_infinite_kl(V):
    """An action that is not allowed, of a finite log-probability under the reference policy, and one the other way round."""
    logits, action, old, adv, ref, _ = loss_data(12, V, torch.float32, 161)
    none = logits.clone()
    none[2, action[2]] = -math.inf
    never = ref.clone()
    never[5] = -math.inf
    for data in ((none, action, old, adv, ref, None), (logits, action, old, adv, never, None)):
        loss, scalars, grad = run_loss(*data, kl_coeff=0.1, **KW)
        assert float(loss) == math.inf and float(scalars[2]) == math.inf
        assert bool(torch.isfinite(scalars[[1, 3, 4]]).all())
        if data[4] is never:                 # e^d - 1 = -1
            _, want = loss64(*data, 0.2, 0.3, 0.1)
            err = (64 + 4) * 2. ** -24 + 2. ** -20         # as in loss_close
            assert bool(((grad.double() - want).abs() <= 2. ** -24 * want.abs()
                         + 4 * err * want.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("V", [7, 18, 100, 500, 3000, 20000, 140000])
def test_policy_kl_loss_without_weight_on_the_kl_term(V):
    """A reference policy that is only watched (kl_coeff = 0): where e^d is beyond 32 bits, kl is infinite, the loss and its
    gradient are those without a reference policy."""
    logits, action, old, adv, ref, w = loss_data(12, V, torch.float32, 160)
    far = ref.clone()
    far[2], w[2] = 100., 1.
    c = dict(entropy_coeff=0.02, **KW)
    loss, scalars, grad = run_loss(logits, action, old, adv, None, w, **c)
    got_loss, got, got_grad = run_loss(logits, action, old, adv, far, w, **c)
    assert torch.equal(got_loss, loss) and torch.equal(got_grad, grad) and float(got[2]) == math.inf
    assert torch.equal(got[[0, 1, 3, 4]], scalars[[0, 1, 3, 4]])
    # an action that is not allowed: log-probability -inf, ratio 0, kl infinite
    none = logits.clone()
    none[2, action[2]] = -math.inf
    loss, scalars, grad = run_loss(none, action, old, adv, None, w, **c)
    got_loss, got, got_grad = run_loss(none, action, old, adv, ref, w, **c)
    assert math.isfinite(float(loss)) and torch.equal(got_loss, loss) and torch.equal(got_grad, grad)
    assert float(got[2]) == math.inf


def test_gated_scan_accuracy_of_the_gates():
    """z from one step out of 0 (h = z x with x = 1), 1 - z from one step out of 1 (x = 0).  In units of 2^-24: the exponent g log2(e) is
    rounded once (|g|) with a rounded factor (0.22 |g|), exp2 2, 1 + e 1, the reciprocal 1, a product 1; in the larger of z and 1 - z the
    exponent's part is weighed down by the smaller."""
    g = torch.linspace(-60., 60., 1 << 16, device=DEV).view(1, 1, -1)
    one, zero = torch.ones_like(g), torch.zeros_like(g)
    for got, want in ((ops.gated_scan(one, g, zero[0])[0], torch.sigmoid(g.double())),
                      (ops.gated_scan(zero, g, one[0])[0], torch.sigmoid(-g.double()))):
        units = torch.where(want >= 0.5, 5., 1.3 * g.abs() + 5.)
        assert bool(((got.double() / want - 1.).abs() <= units.double() * 2. ** -24).all())


def test_orthogonalize_does_not_depend_on_the_run():
    """Products split over their sums among them, and memory that holds something else each time."""
    for sizes, dtype in ((((512, 3456), (18, 512), (32, 256)), torch.float32), (((1601, 1700),), torch.bfloat16)):
        mats = [torch.randn(*s, device=DEV, generator=gen(170)).to(dtype) for s in sizes]
        first = ops.orthogonalize(mats)
        for k in range(3):
            torch.full((1 << 26,), math.nan, device=DEV)          # (freed at once: the next workspace lies there)
            ops.orthogonalize([m + k + 1 for m in mats])
            assert all(torch.equal(a, b) for a, b in zip(ops.orthogonalize(mats), first))


@pytest.mark.parametrize("V", [18, 100, 500, 3000, 20000, 140000])
def test_policy_kl_loss_weights_of_any_sign(V):
    """The mean divides by the sum of the weights, whatever its sign; a NaN among them shows in the gradient too."""
    logits, action, old, adv, ref, w = loss_data(14, V, torch.float32, 162)
    w = torch.where(torch.arange(14, device=DEV) % 3 == 0, 0.25 * (w + 0.1), -(w + 0.1))
    w[4] = 0.
    c = dict(kl_coeff=0.1, entropy_coeff=0.02)
    out = run_loss(logits, action, old, adv, ref, w, **KW, **c)
    want_s, want_g = loss64(logits, action, old, adv, ref, w, 0.2, 0.3, 0.1, 0.02)
    err = 4 * ((64 + 4) * 2. ** -24 + 2. ** -20)         # as in loss_close, of the terms, which cancel here by as much as the weights do
    cancel = float(w.double().abs().sum() / w.double().sum().abs())
    assert bool(((out[1].double() - want_s).abs() <= err * cancel * (want_s.abs().max() + 4 * math.log(V))).all()), (out[1], want_s)
    assert bool(((out[2].double() - want_g).abs() <= err * want_g.abs().amax(-1, keepdim=True)).all())
    same = run_loss(logits, action, old, adv, ref, -w, **KW, **c)
    assert torch.equal(same[1], out[1]) and torch.equal(same[2], out[2])
    w[5] = math.nan
    loss, _, grad = run_loss(logits, action, old, adv, ref, w, **KW, **c)
    assert math.isnan(float(loss)) and bool(torch.isnan(grad[w != 0]).all()) and not bool(grad[4].any())
