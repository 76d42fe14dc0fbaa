"""Refusals of the sequence operators (no GPU needed): wrong shapes, types and options raise before any device
call, and the C entry points return error codes with a message."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest
import torch

from rlpyt_amd import _lib, ops
from rlpyt_amd.optim import Muon

z = torch.zeros


@pytest.mark.parametrize("call", [
    lambda: ops.gated_scan(z(3, 2), z(3, 2)),                                       # not [T, B, D]
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 5)),
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4).bfloat16()),                      # two types
    lambda: ops.gated_scan(z(3, 2, 4).double(), z(3, 2, 4).double()),
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4), h0=z(4, 2)),
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4), h0=z(2, 4).long()),
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4), reset=z(2, 3).bool()),
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4), lengths=z(2)),                   # not whole numbers
    lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4), lengths=z(3).long()),
    lambda: ops.gated_scan_step(z(2, 4), z(4, 2), z(2, 4)),
    lambda: ops.gated_scan_step(z(2, 4), z(2, 4), z(2, 4).bfloat16()),              # the state is float32
    lambda: ops.gated_scan_step(z(2, 4), z(2, 4), z(4, 2).t()),                     # and dense
    lambda: ops.gated_scan_step(z(2, 4), z(2, 4), z(2, 4), reset=z(4).bool()),
    lambda: ops.gated_scan_step(z(2, 4, requires_grad=True), z(2, 4), z(2, 4)),
    lambda: ops.policy_kl_loss(z(3, 0), z(3).long(), z(3), z(3)),
    lambda: ops.policy_kl_loss(z(3, 4).double(), z(3).long(), z(3), z(3)),
    lambda: ops.policy_kl_loss(z(3, 4), z(3), z(3), z(3)),                          # action not whole
    lambda: ops.policy_kl_loss(z(3, 4), z(4).long(), z(3), z(3)),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(4), z(3)),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(1)),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), valid=z(3, 1)),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), kl_coeff=0.1),     # no ref_logp
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), clip_low=1.5),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), clip_high=-0.1),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), clip_high=float("nan")),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), grad_scale=0.),
    lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3), grad_scale=float("inf")),
    lambda: ops.action_logp(z(3, 4), z(3)),
    lambda: ops.action_logp(z(3, 4).long(), z(3).long()),
    lambda: ops.orthogonalize(z(4)),
    lambda: ops.orthogonalize([z(4, 4), z(4, 4).double()]),
    lambda: ops.orthogonalize(z(4, 4), steps=0),
    lambda: ops.orthogonalize(z(4, 4), steps=2.5),
    lambda: ops.orthogonalize(z(4, 4), coeffs=(1., 2.)),
    lambda: ops.orthogonalize(z(4, 4), eps=-1.),
    lambda: ops.gated_scan(z(1, 1, 1).expand(1, 1 << 15, 1 << 14), z(1, 1, 1).expand(1, 1 << 15, 1 << 14)),
    lambda: ops.gated_scan(z(1, 1, 1).expand(1 << 30, 1, 1), z(1, 1, 1).expand(1 << 30, 1, 1)),
    lambda: ops.gated_scan_step(z(1, 1).expand(1 << 15, 1 << 14), z(1, 1).expand(1 << 15, 1 << 14), z(1, 1)),
    lambda: ops.policy_kl_loss(z(1, 1).expand(1, (1 << 30) + 1), z(1).long(), z(1), z(1)),
    lambda: ops.action_logp(z(1, 1).expand(1, (1 << 30) + 1), z(1).long()),
    lambda: ops.orthogonalize(z(1, 1).expand(1, (1 << 16) + 1)),
    lambda: Muon([z(3, 3, requires_grad=True)], lr=-1.),
    lambda: Muon([z(3, 3, requires_grad=True)], momentum=1.),
])
def test_refused(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="GPU present")
def test_no_cpu_fallback():
    for call in (lambda: ops.gated_scan(z(3, 2, 4), z(3, 2, 4)), lambda: ops.gated_scan_step(z(2, 4), z(2, 4), z(2, 4)),
                 lambda: ops.policy_kl_loss(z(3, 4), z(3).long(), z(3), z(3)),
                 lambda: ops.action_logp(z(3, 4), z(3).long()), lambda: ops.orthogonalize(z(4, 4))):
        with pytest.raises(_lib.HipError):
            call()


def test_orthogonalize_of_nothing():
    assert ops.orthogonalize([]) == []


def test_entry_points_validate_without_a_gpu():
    lib = _lib.lib
    buf = (ctypes.c_float * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    fwd, bwd = lib.rlpyt_gated_scan_fwd, lib.rlpyt_gated_scan_bwd
    # nothing to do
    assert fwd(0, None, 0, 0, None, 0, 0, None, None, None, None, 0, 0, None, None, 0, 2, 4, None, None) == 0
    assert bwd(0, None, 0, 0, None, 0, 0, None, 0, 0, None, None, None, None, None, 0, 0, None, 0, 0, None, 3, 0, 4,
               None, None) == 0
    # unknown type, sizes out of range, null pointers
    assert fwd(3, p, 0, 0, p, 0, 0, None, None, None, p, 0, 0, None, None, 1, 1, 4, None, None) != 0
    assert b"dtype" in lib.rlpyt_hip_last_error()
    assert fwd(0, p, 0, 0, p, 0, 0, None, None, None, p, 0, 0, None, None, -1, 1, 4, None, None) != 0
    assert fwd(0, p, 0, 0, p, 0, 0, None, None, None, p, 0, 0, None, None, 1, 1 << 20, 1 << 20, None, None) != 0
    assert b"out of range" in lib.rlpyt_hip_last_error()
    assert fwd(0, None, 0, 0, p, 0, 0, None, None, None, p, 0, 0, None, None, 1, 1, 4, None, None) != 0
    assert b"null pointer" in lib.rlpyt_hip_last_error()
    # a long sequence of few channels needs its workspace
    assert lib.rlpyt_gated_scan_workspace_bytes(1 << 16, 1, 512) > 0
    assert fwd(0, p, 0, 0, p, 0, 0, None, None, None, p, 0, 0, None, None, 1 << 16, 1, 512, None, None) != 0
    assert b"workspace" in lib.rlpyt_hip_last_error()
    assert lib.rlpyt_gated_scan_workspace_bytes(0, 1, 512) == 0
    assert lib.rlpyt_gated_scan_state_rows(0) == 0 and lib.rlpyt_gated_scan_state_rows(1) == 1
    assert lib.rlpyt_gated_scan_step(0, None, 0, None, 0, None, None, None, 0, 4, None) == 0
    assert lib.rlpyt_gated_scan_step(0, None, 0, None, 0, None, None, None, 2, 4, None) != 0
    loss = lib.rlpyt_policy_kl_loss_fwd_bwd
    assert loss(0, p, 4, p, p, p, None, None, 2, 0, .2, .2, 0., 0., 1., p, p, None, p, None) != 0
    assert loss(0, None, 4, p, p, p, None, None, 2, 4, .2, .2, 0., 0., 1., p, p, None, p, None) != 0
    assert loss(0, p, 4, p, p, p, None, None, 2, 4, .2, .2, 0., 0., 1., None, p, None, p, None) != 0
    assert loss(0, p, 4, p, p, p, None, None, 2, 4, .2, .2, 0., 0., 1., p, p, None, None, None) != 0
    assert lib.rlpyt_action_logp(0, None, 4, None, 0, 4, None, None, None, None) == 0
    assert lib.rlpyt_action_logp(0, None, 4, None, 2, 4, None, None, None, None) != 0
    assert lib.rlpyt_scale_unless_one(0, None, 0, None, 1., None) == 0
    assert lib.rlpyt_scale_unless_one(0, None, 4, None, 1., None) != 0
    one = (ctypes.c_void_p * 1)(p.value)
    side, big = (ctypes.c_int64 * 1)(4), (ctypes.c_int64 * 1)(1 << 20)
    orth = lib.rlpyt_orthogonalize
    assert orth(0, None, None, None, None, None, 0, 5, 1., 0., 0., 0., None, None) == 0
    assert orth(0, one, side, one, big, side, 1, 5, 1., 0., 0., 0., p, None) != 0
    assert orth(0, one, side, one, side, side, 1, 5, 1., 0., 0., 0., None, None) != 0
    assert orth(0, one, side, one, side, side, 1, 5, 9., 0., 0., 0., p, None) != 0     # leaves f16's range
    assert b"range of the stored factors" in lib.rlpyt_hip_last_error()
    assert orth(0, one, side, one, side, side, 1, 5, float("nan"), 0., 0., 0., p, None) != 0


LOSS_PLAN = r"""
#include <cstdint>
#include <cstdio>
namespace rlpyt { static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; } }
#include "policy_loss_plan.h"
int main() {
  using namespace rlpyt;
  int bad = 0;
  for (int size : {2, 4})
    for (int64_t V : {1, 5, 128, 129, 4096, 4097, 32768, 32769, 65536, 65537, 131072, 131073, 300007, 1 << 30})
      for (int64_t N : {0, 1, 3, 127, 128, 1023, 1025, 32768, 3000000}) {
        const LossPlan q = plan_of(N, V, size);
        const int64_t slice = slice_rows(q);
        // parts that cover a row, none of them empty or off a 16-byte step; a launch of less than 2^32 threads
        bool ok = q.P >= 0 && slice > 0 && slice * (q.P > 0 ? q.P * 256 : 1024) < (int64_t)1 << 32;
        if (q.P > 0) ok = ok && q.part % 8 == 0 && (int64_t)q.part * q.P >= V && (int64_t)q.part * (q.P - 1) < V;
        if (N == 0) ok = ok && q.groups(0) == 0;
        if (!ok) ++bad, printf("N %ld V %ld size %d: P %d part %d\n", (long)N, (long)V, size, q.P, q.part);
      }
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_plan_of_the_policy_loss(tmp_path):
    """Compiled on its own and unoptimised: an optimiser may drop a division by zero, the machine does not."""
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(LOSS_PLAN)
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    subprocess.run(["g++", "-std=c++17", "-O0", "-I", csrc, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stdout)


@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_derivatives_are_refused(needs_grad):
    """A dual tensor does not require a gradient by itself; its derivative must not get lost."""
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        def dual(*shape):
            return fw.make_dual(z(*shape, requires_grad=needs_grad), torch.ones(*shape))

        seq, row, one = z(3, 2, 4), z(2, 4), z(3)
        calls = [
            lambda: ops.gated_scan(dual(3, 2, 4), seq), lambda: ops.gated_scan(seq, dual(3, 2, 4)),
            lambda: ops.gated_scan(seq, seq, h0=dual(2, 4)),
            lambda: ops.policy_kl_loss(dual(3, 4), one.long(), one, one),
            lambda: ops.policy_kl_loss(z(3, 4), one.long(), dual(3), one),
            lambda: ops.policy_kl_loss(z(3, 4), one.long(), one, dual(3)),
            lambda: ops.policy_kl_loss(z(3, 4), one.long(), one, one, ref_logp=dual(3)),
            lambda: ops.policy_kl_loss(z(3, 4), one.long(), one, one, valid=dual(3)),
            lambda: ops.action_logp(dual(3, 4), one.long()),
            lambda: ops.orthogonalize(dual(4, 4)), lambda: ops.orthogonalize([z(4, 4), dual(2, 4, 4)]),
        ]
        steps = [lambda: ops.gated_scan_step(dual(2, 4), row, row), lambda: ops.gated_scan_step(row, dual(2, 4), row),
                 lambda: ops.gated_scan_step(row, row, dual(2, 4))]
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        for call in steps:
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):     # (this mode goes on under no_grad)
                call()


@pytest.mark.parametrize("call", [
    lambda t: ops.action_logp(t, z(4).long()), lambda t: ops.orthogonalize(t), lambda t: ops.orthogonalize([z(3, 3), t]),
])
def test_gradients_that_would_be_lost_are_refused(call):
    with pytest.raises(ValueError, match="not differentiable"):
        call(z(4, 4, requires_grad=True))
    with torch.no_grad(), pytest.raises((ValueError, _lib.HipError), match="device|MI355X"):     # (these are on the CPU)
        call(z(4, 4, requires_grad=True))


def optimizer_of(algo):
    params = [torch.nn.Parameter(z(3, 4)), torch.nn.Parameter(z(3))]
    return algo.make_optimizer(params, algo.OptimCls, algo.learning_rate, algo.optim_kwargs)


@pytest.mark.parametrize("given", [None, dict(momentum=0.5)])
def test_algorithms_build_muon(given):
    """Also those whose defaults are Adam's: its eps goes to the optimizers that have one."""
    from rlpyt_amd.algos.dqn.cat_dqn import CategoricalDQN
    from rlpyt_amd.algos.dqn.dqn import DQN
    from rlpyt_amd.algos.dqn.r2d1 import R2D1
    from rlpyt_amd.algos.pg.a2c import A2C
    from rlpyt_amd.algos.pg.ppo import PPO
    for Algo in (PPO, A2C, DQN, CategoricalDQN, R2D1):
        kwargs = None if given is None else dict(given)
        opt = optimizer_of(Algo(OptimCls=Muon, optim_kwargs=kwargs, learning_rate=0.02))
        assert type(opt) is Muon and opt.param_groups[0]["momentum"] == (0.95 if given is None else 0.5)
        assert kwargs == given                      # the caller's own dict stays as it was
    for Algo, eps in ((DQN, 0.01 / 32), (CategoricalDQN, 0.01 / 32), (R2D1, 1e-3)):
        for OptimCls in (torch.optim.Adam, torch.optim.AdamW, torch.optim.RMSprop):
            assert optimizer_of(Algo(OptimCls=OptimCls)).param_groups[0]["eps"] == eps
            assert optimizer_of(Algo(OptimCls=OptimCls, optim_kwargs=dict(eps=0.5))).param_groups[0]["eps"] == 0.5
        assert "eps" not in optimizer_of(Algo(OptimCls=torch.optim.SGD)).param_groups[0]


@pytest.mark.parametrize("max_norm", [None, 0., -1., float("inf")])
def test_muon_without_a_bound_leaves_the_gradients(max_norm):
    """An infinite gradient then stays in its own parameter; what is returned is the norm."""
    a, b = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    a.grad, b.grad = torch.full((3,), 2.), torch.tensor([1., float("inf"), 1.])
    norm = Muon([a, b], lr=0.02).clip_and_step(max_norm)
    assert float(norm) == float("inf")
    assert torch.equal(a.grad, torch.full((3,), 2.))
    assert torch.allclose(a.detach(), torch.full((3,), 0.999))         # Adam's first step: lr x adam_lr_ratio
    b.grad = torch.tensor([1., 2., 2.])
    norm = Muon([a, b], lr=0.02).clip_and_step(max_norm)
    assert abs(float(norm) - 21 ** 0.5) < 1e-6 and torch.equal(b.grad, torch.tensor([1., 2., 2.]))
    norm = Muon([a, b], lr=0.02).clip_and_step(1.)
    assert abs(float(norm) - 21 ** 0.5) < 1e-6 and abs(float(torch.cat([a.grad, b.grad]).norm()) - 1.) < 1e-5


WITHOUT_EXTENSION = """
import sys, types
class Gone:
    def find_spec(self, name, path=None, target=None):
        if name == "rlpyt_amd._seqops":
            raise ImportError("undefined symbol: of another torch")
sys.meta_path.insert(0, Gone())
from rlpyt_amd import _lib, ops, ops_seq, optim
from rlpyt_amd.algos.dqn.r2d1 import R2D1
from rlpyt_amd.algos.pg.ppo import PPO
assert ops.orthogonalize([]) == [] and callable(ops.gae)
stale = types.ModuleType("rlpyt_amd._seqops")
stale.abi_version = _lib.ABI_VERSION - 1
for wrong in ("cannot be loaded", "cannot be loaded", "rebuild"):
    if wrong == "rebuild":
        sys.modules["rlpyt_amd._seqops"] = stale
    for use in (lambda: ops_seq._seqops.gated_scan, lambda: ops_seq._seqops.action_logp):
        try:
            use()
        except _lib.HipExtensionMissing as e:
            assert wrong in str(e), e
        else:
            raise SystemExit("used without the extension")
"""


def test_only_the_operators_that_use_the_extension_need_it():
    """The rest of the package imports where ``_seqops.so`` is missing or was built against another torch; the operators behind
    it fail loudly, every time."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
    run = subprocess.run([sys.executable, "-c", WITHOUT_EXTENSION], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("options", [dict(coeffs=(9., 0., 0.)), dict(coeffs=(3., 0., 3.)), dict(coeffs=(float("nan"), 0., 0.)),
                                     dict(coeffs=(2., float("inf"), 0.)), dict(steps=float("inf")), dict(steps=float("nan"))])
def test_orthogonalize_refuses_its_options_as_arguments(options):
    """As ValueError like every argument that does not fit, and first of all: before the matrices are looked at."""
    for mats in (z(4, 4), [z(4, 4), z(2, 3, 5)], []):
        with pytest.raises(ValueError):
            ops.orthogonalize(mats, **options)


def test_orthogonalize_takes_bounded_options():
    for steps, coeffs in ((5, (3.4445, -4.7750, 2.0315)), (100, (1.5, -0.5, 0.)), (3., (2., -1.5, 0.5))):
        assert ops.orthogonalize([], steps=steps, coeffs=coeffs) == []


@pytest.mark.parametrize("T,channels,split", [
    (64, 1, False), (85, 16 * 512, False), (128, 16 * 512, False), (192, 64, False), (256, 64, True), (256, 64 * 64, True),
    (448, 80 * 64, False), (512, 80 * 64, True), (960, 112 * 64, False), (1024, 112 * 64, True), (1 << 16, 128 * 64, True),
    (2048, 144 * 64, False), (1 << 16, 160 * 64, False), (1 << 16, 512, True),
])
def test_where_time_is_split(T, channels, split):
    """Segments of time (whose maps are the workspace) need steps enough to pay for their launch and their second read."""
    assert (_lib.lib.rlpyt_gated_scan_workspace_bytes(T, channels, 1) > 0) == split    # D = 1: 64 channels a tile in every type
