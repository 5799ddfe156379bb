"""Refusals of the token, normalisation and fine-tuning operators: what the Python entry points and the C ABI reject before
any kernel is launched.  None of these needs a GPU: the C calls below are refused from their sizes and flags, and the address
they pass is never dereferenced."""
import ctypes

import pytest
import torch

from graphmaker_amd import _lib as L
from graphmaker_amd import autograd as ag

P = ctypes.addressof(ctypes.create_string_buffer(64)) // 16 * 16 + 16      # a non-null aligned address nobody reads
BIG = 1 << 31


def f(*shape, dtype=torch.float32, grad=False):
    return torch.zeros(*shape, dtype=dtype, requires_grad=grad)


def i(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call, error", [
    (lambda: ag.token_embedding(f(4), i(3)), ValueError),
    (lambda: ag.token_embedding(f(0, 4), i(3)), ValueError),
    (lambda: ag.token_embedding(f(4, 0), i(3)), ValueError),
    (lambda: ag.token_embedding(f(4, 8, dtype=torch.float64), i(3)), TypeError),
    (lambda: ag.token_embedding(f(4, 8), i(3, dtype=torch.int16)), TypeError),
    (lambda: ag.token_embedding(f(4, 8), f(3)), TypeError),
    (lambda: ag.token_embedding(f(4, 8), i(3), padding_idx=4), ValueError),
    (lambda: ag.token_embedding(f(4, 8), i(3), padding_idx=-5), ValueError),
    (lambda: ag.token_embedding(f(4, 8), i(3), scale=float("inf")), ValueError),
    (lambda: ag.token_embedding(f(4, 8), i(3), scale=1e39), ValueError),
    (lambda: ag.token_embedding(f(4, 8), i(3)), L.GraphMakerHipError),
    (lambda: ag.layer_norm(f(())), ValueError),
    (lambda: ag.layer_norm(f(3, 0)), ValueError),
    (lambda: ag.layer_norm(f(3, 4, dtype=torch.float64)), TypeError),
    (lambda: ag.layer_norm(f(3, 4), f(5)), ValueError),
    (lambda: ag.layer_norm(f(3, 4), f(4), f(1, 4)), ValueError),
    (lambda: ag.layer_norm(f(3, 4), f(4, dtype=torch.bfloat16)), TypeError),
    (lambda: ag.layer_norm(f(3, 4, dtype=torch.bfloat16), f(4), f(4, dtype=torch.bfloat16)), TypeError),
    (lambda: ag.layer_norm(f(3, 4, dtype=torch.bfloat16), f(4, dtype=torch.float16)), TypeError),
    (lambda: ag.layer_norm(f(3, 4), eps=-1e-5), ValueError),
    (lambda: ag.layer_norm(f(3, 4), eps=float("nan")), ValueError),
    (lambda: ag.layer_norm(f(3, 4), f(4), f(4)), L.GraphMakerHipError),
    (lambda: ag.class_log_prob(f(()), i(())), ValueError),
    (lambda: ag.class_log_prob(f(3, 0), i(3)), ValueError),
    (lambda: ag.class_log_prob(f(3, 4), i(3, 1)), ValueError),
    (lambda: ag.class_log_prob(f(3, 4, dtype=torch.float64), i(3)), TypeError),
    (lambda: ag.class_log_prob(f(3, 4), i(3, dtype=torch.uint8)), TypeError),
    (lambda: ag.class_log_prob(f(3, 4), i(3)), L.GraphMakerHipError),
])
def test_row_operators_refuse(call, error):
    with pytest.raises(error):
        call()


def _policy(**kw):
    a = dict(log_prob=f(6), old_log_prob=f(6), advantage=f(6))
    a.update(kw)
    return ag.policy_loss(a.pop("log_prob"), a.pop("old_log_prob"), a.pop("advantage"), **a)


@pytest.mark.parametrize("kw, error", [
    (dict(log_prob=f(6, dtype=torch.float16)), TypeError),
    (dict(old_log_prob=f(5)), ValueError),
    (dict(old_log_prob=f(6, dtype=torch.float64)), TypeError),
    (dict(old_log_prob=f(6, grad=True)), ValueError),
    (dict(advantage=f(6, grad=True)), ValueError),
    (dict(advantage=f(2)), ValueError),
    (dict(ref_log_prob=f(6, grad=True)), ValueError),
    (dict(ref_log_prob=f(6, 1)), ValueError),
    (dict(mask=f(6)), TypeError),
    (dict(mask=torch.ones(5, dtype=torch.bool)), ValueError),
    (dict(offsets=i(1), advantage=f(0)), ValueError),
    (dict(offsets=i(2, 2)), ValueError),
    (dict(offsets=f(3), advantage=f(2)), TypeError),
    (dict(offsets=i(3)), ValueError),
    (dict(offsets=i(3), advantage=f(2, grad=True)), ValueError),
    (dict(reduction="mean"), ValueError),
    (dict(reduction="sequence"), ValueError),
    (dict(clip_low=1.5), ValueError),
    (dict(clip_low=-0.1), ValueError),
    (dict(clip_high=-0.1), ValueError),
    (dict(clip_high=float("nan")), ValueError),
    (dict(kl_coef=0.1), ValueError),
    (dict(kl_coef=float("inf"), ref_log_prob=f(6)), ValueError),
    (dict(), L.GraphMakerHipError),
])
def test_policy_loss_refuses(kw, error):
    with pytest.raises(error):
        _policy(**kw)


@pytest.mark.parametrize("args, kw, error", [
    ((f(6), f(6), i(2)), {}, ValueError),                  # one sequence
    ((f(6), f(6), i(4)), {}, ValueError),                  # three
    ((f(6), f(6), i(1)), {}, ValueError),
    ((f(6), f(5), i(3)), {}, ValueError),
    ((f(6), f(6, grad=True), i(3)), {}, ValueError),
    ((f(6, dtype=torch.bfloat16), f(6), i(3)), {}, TypeError),
    ((f(6), f(6), i(3, dtype=torch.int16)), {}, TypeError),
    ((f(6), f(6), i(3)), dict(mask=i(6)), TypeError),
    ((f(6), f(6), i(3)), dict(beta=0.0), ValueError),
    ((f(6), f(6), i(3)), dict(beta=float("inf")), ValueError),
    ((f(6), f(6), i(3)), dict(label_smoothing=0.6), ValueError),
    ((f(6), f(6), i(3)), dict(label_smoothing=-0.1), ValueError),
    ((f(6), f(6), i(3)), {}, L.GraphMakerHipError),
])
def test_preference_loss_refuses(args, kw, error):
    with pytest.raises(error):
        ag.preference_loss(*args, **kw)


@pytest.mark.parametrize("name, args", [
    ("gm_token_embedding_fwd", (-1, 4, 8, P, 0, P, 8, 0, 1.0, P, 8)),
    ("gm_token_embedding_fwd", (3, 0, 8, P, 0, P, 8, 0, 1.0, P, 8)),
    ("gm_token_embedding_fwd", (3, 4, 8, P, 0, P, 7, 0, 1.0, P, 8)),
    ("gm_token_embedding_fwd", (3, 4, 8, P, 0, P, 8, 0, 1.0, P, 7)),
    ("gm_token_embedding_fwd", (3, 4, 8, P, 0, P, 8, 3, 1.0, P, 8)),
    ("gm_token_embedding_fwd", (3, 4, 8, None, 0, P, 8, 0, 1.0, P, 8)),
    ("gm_token_embedding_fwd", (BIG, 4, 8, P, 0, P, 8, 0, 1.0, P, 8)),
    ("gm_token_embedding_bwd", (3, 4, 8, P, 0, 4, P, 8, 0, 1.0, P, 8, P, 1 << 20)),
    ("gm_token_embedding_bwd", (3, 4, 8, P, 0, -1, P, 8, 0, 1.0, P, 8, P, 16)),
    ("gm_token_embedding_bwd", (3, 4, 8, P, 0, -1, P, 8, 0, 1.0, P, 8, None, 1 << 20)),
    ("gm_token_embedding_bwd", (3, 4, 8, P, 0, -1, P, 8, 0, 1.0, None, 8, P, 1 << 20)),
    ("gm_token_embedding_bwd", (3, 4, 8, P, 0, -1, P, 7, 0, 1.0, P, 8, P, 1 << 20)),
    ("gm_layer_norm_fwd", (3, 0, P, 8, 0, P, P, 0, 1e-5, P, 8, P, P)),
    ("gm_layer_norm_fwd", (3, 8, P, 7, 0, P, P, 0, 1e-5, P, 8, P, P)),
    ("gm_layer_norm_fwd", (3, 8, P, 8, 1, P, P, 2, 1e-5, P, 8, P, P)),
    ("gm_layer_norm_fwd", (3, 8, P, 8, 0, P, P, 1, 1e-5, P, 8, P, P)),
    ("gm_layer_norm_fwd", (3, 8, P, 8, 0, P, P, 0, 1e-5, P, 8, P, None)),
    ("gm_layer_norm_fwd", (BIG, 8, P, 8, 0, P, P, 0, 1e-5, P, 8, P, P)),
    ("gm_layer_norm_bwd", (3, 8, P, 8, P, 8, 0, P, P, P, 0, P, 8, P, P, P, 8)),
    ("gm_layer_norm_bwd", (3, 8, P, 8, P, 8, 0, P, P, P, 0, P, 8, P, P, None, 1 << 20)),
    ("gm_layer_norm_bwd", (3, 8, P, 8, P, 8, 0, None, P, P, 0, P, 8, None, None, None, 0)),
    ("gm_layer_norm_bwd", (3, 8, P, 8, P, 8, 0, P, P, P, 0, P, 7, None, None, None, 0)),
    ("gm_class_log_prob_fwd", (3, 8, P, 7, 0, P, 0, -100, P, P, None, 0)),
    ("gm_class_log_prob_fwd", (3, 8, P, 8, 5, P, 0, -100, P, P, None, 0)),
    ("gm_class_log_prob_fwd", (3, 8, P, 8, 0, None, 0, -100, P, P, None, 0)),
    ("gm_class_log_prob_fwd", (3, BIG, P, BIG, 0, P, 0, -100, P, P, None, 0)),
    ("gm_class_log_prob_bwd", (3, 8, P, P, 8, 0, P, 0, -100, P, P, 7)),
    ("gm_class_log_prob_bwd", (3, 8, None, P, 8, 0, P, 0, -100, P, P, 8)),
    ("gm_class_log_prob_bwd", (3, 8, P, P, 8, 0, P, 0, -100, P, None, 8)),
    ("gm_policy_loss_fwd", (3, 0, P, P, P, None, None, P, 0, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 20)),
    ("gm_policy_loss_fwd", (3, 2, P, P, P, None, None, None, 0, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 20)),
    ("gm_policy_loss_fwd", (3, 1, P, P, P, None, None, P, 0, 0.2, 0.2, 0.1, 0, P, P, P, P, P, 1 << 20)),
    ("gm_policy_loss_fwd", (3, 1, P, P, P, None, None, P, 0, 1.2, 0.2, 0.0, 0, P, P, P, P, P, 1 << 20)),
    ("gm_policy_loss_fwd", (3, 1, P, P, P, None, None, P, 0, 0.2, float("nan"), 0.0, 0, P, P, P, P, P, 1 << 20)),
    ("gm_policy_loss_fwd", (3, 1, P, P, P, None, None, P, 0, 0.2, 0.2, 0.0, 0, P, P, P, P, P, 8)),
    ("gm_policy_loss_fwd", (3, 1, P, P, P, None, None, P, 0, 0.2, 0.2, 0.0, 0, None, P, P, P, P, 1 << 20)),
    ("gm_preference_loss_fwd", (3, 0, P, P, None, P, 0, 0.1, 0.0, 0, P, P, P, P, 1 << 20)),
    ("gm_preference_loss_fwd", (3, 1, P, P, None, None, 0, 0.1, 0.0, 0, P, P, P, P, 1 << 20)),
    ("gm_preference_loss_fwd", (3, 1, P, P, None, P, 0, 0.0, 0.0, 0, P, P, P, P, 1 << 20)),
    ("gm_preference_loss_fwd", (3, 1, P, P, None, P, 0, 0.1, 0.7, 0, P, P, P, P, 1 << 20)),
    ("gm_preference_loss_fwd", (3, 1, P, P, None, P, 0, 0.1, 0.0, 0, P, P, P, P, 8)),
    ("gm_sequence_loss_bwd", (3, 0, P, None, P, 0, P, P, P)),
    ("gm_sequence_loss_bwd", (3, 2, P, None, None, 0, P, P, P)),
    ("gm_sequence_loss_bwd", (3, 1, P, None, P, 0, None, P, P)),
])
def test_c_entry_points_refuse(name, args):
    lib = L.load()
    assert getattr(lib, name)(*args, None) == -1, "not refused"               # GM_E_INVALID
    assert lib.gm_last_error()


def test_workspace_sizes():
    lib = L.load()
    assert lib.gm_token_embedding_bwd_workspace_bytes(0, 5, 8) > 0
    assert lib.gm_token_embedding_bwd_workspace_bytes(-1, 5, 8) == -1
    assert lib.gm_token_embedding_bwd_workspace_bytes(BIG, 5, 8) == -1
    assert lib.gm_layer_norm_bwd_workspace_bytes(0, 8) >= 0
    assert lib.gm_layer_norm_bwd_workspace_bytes(8, 0) == -1 == lib.gm_layer_norm_bwd_workspace_bytes(8, 1 << 26)
    assert lib.gm_class_log_prob_stats_floats(8, 1 << 28, 1) == -1 == lib.gm_sequence_loss_workspace_bytes(1 << 34, 1)
    assert lib.gm_class_log_prob_stats_floats(1, 1 << 27, 0) == -1 == lib.gm_class_log_prob_workspace_bytes(1, 1 << 27, 0)
    assert lib.gm_class_log_prob_workspace_bytes(8, 0, 0) == -1 == lib.gm_class_log_prob_workspace_bytes(8, 8, 3)
    assert lib.gm_class_log_prob_stats_floats(8, 3, 0) == 0 and lib.gm_class_log_prob_stats_floats(8, 4, 0) == 16
    assert lib.gm_class_log_prob_stats_floats(8, 7, 1) == 0 and lib.gm_class_log_prob_stats_floats(8, 8, 1) == 16
    assert lib.gm_class_log_prob_stats_floats(8, 8, -1) == -1
    assert lib.gm_sequence_loss_workspace_bytes(8, 0) == -1
    assert lib.gm_sequence_loss_workspace_bytes(0, 1) > 0


def test_signatures_match_the_header():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "graphmaker_hip.h")).read()
    for name, kinds in L._SIGNATURES.items():
        args = re.search(r"\b" + name + r"\(([^)]*)\)", header, re.S).group(1).split(",")
        want = "".join("p" if "*" in a or "gm_stream_t" in a else "i" if "int64_t" in a else "f" if "float" in a else "d" for a in args)
        assert kinds == want, name


def dual(t):
    import torch.autograd.forward_ad as fwd
    return fwd.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("call", [
    lambda: ag.token_embedding(dual(f(4, 8)), i(3)),
    lambda: ag.layer_norm(dual(f(3, 4)), f(4), f(4)),
    lambda: ag.layer_norm(f(3, 4), dual(f(4)), f(4)),
    lambda: ag.layer_norm(f(3, 4), None, dual(f(4))),
    lambda: ag.layer_norm(dual(f(3, 4)), f(4, grad=True), f(4)),
    lambda: ag.class_log_prob(dual(f(3, 4)), i(3)),
    lambda: ag.policy_loss(dual(f(6)), f(6), f(6)),
    lambda: ag.policy_loss(f(6, grad=True), dual(f(6)), f(6)),
    lambda: ag.policy_loss(f(6), f(6), dual(f(6))),
    lambda: ag.policy_loss(f(6), f(6), dual(f(2)), offsets=i(3)),
    lambda: ag.policy_loss(f(6), f(6), f(6), ref_log_prob=dual(f(6))),
    lambda: ag.preference_loss(dual(f(6)), f(6), i(3)),
    lambda: ag.preference_loss(f(6), dual(f(6)), i(3)),
])
def test_forward_mode_derivatives_are_refused(call):
    """An output without a tangent would count as a derivative of zero; the package's other operators raise this error too."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        call()
