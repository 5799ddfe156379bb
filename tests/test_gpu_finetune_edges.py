"""GPU tests at the edges of the fine-tuning operators, against definitions in float64 on the CPU: values past float32 inside a
loss, NaN that must show, gradients of unlikely classes, what a call keeps alive, and rows at any place.

Tolerances count roundings; U = 2^-24 is half a step of float32.
"""
import math

import pytest
import torch

from graphmaker_amd import autograd as ag
from test_gpu_finetune import DT, TYPES, U, check_norm, close, ratios, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("offsets", [None, [0, 15, 40]])
def test_policy_loss_shows_nan_at_advantage_zero(dev, offsets):
    """A log-probability of NaN (a class outside the table) shows whatever its advantage, as r * 0 does; a masked one never."""
    M, at = 40, 7
    lp, old, _ = ratios(3, M)
    adv = torch.tensor([0.0, 1.0]) if offsets else torch.arange(M).float() - at
    kw = dict(offsets=torch.tensor(offsets, device=dev)) if offsets else {}

    def run(lp, old, **more):
        a = lp.to(dev).requires_grad_(True)
        loss, stats = ag.policy_loss(a, old.to(dev), adv.to(dev), **kw, **more)
        return loss.detach(), stats, torch.autograd.grad(loss, [a])[0]

    want = run(lp, old)
    assert all(t.isfinite().all() for t in want) and want[2][at] == 0
    for x, y in ((math.nan, -1.0), (-1.0, math.nan), (-1.0, -math.inf)):         # the last: a ratio of inf times 0
        bad, bad_old = lp.clone(), old.clone()
        bad[at], bad_old[at] = x, y
        loss, stats, dl = run(bad, bad_old)
        assert loss.isnan() and stats[0].isnan() and stats[2:].isfinite().all()
        assert dl[at].isnan() and dl[torch.arange(M, device=dev) != at].isfinite().all()
        mask = torch.arange(M, device=dev) != at
        assert all(t.isfinite().all() for t in run(bad, bad_old, mask=mask))
    for x, y in ((-math.inf, -1.0), (-1.0, -300.0), (-1.0, -3000.0)):            # a ratio of 0, and finite ones of any size
        fine, fine_old = lp.clone(), old.clone()
        fine[at], fine_old[at] = x, y
        for a, b in zip(run(fine, fine_old), want):
            assert torch.equal(a, b)


def policy_formula(lp, old, adv, ref, kl, low=0.2, high=0.28):
    """(loss, stats, gradient) of the mean over all items in float64, and what float32 terms may be off by.

    The ratio and exp(q) are float32: 4 U of the exponential and |x| U of its argument's rounding; one U more of every product,
    sum and border.  Below |q| = 1 exp(q) - 1 - q is a series: 1.2 U left out, 4 U of its own roundings."""
    low, high, kl = (float(torch.tensor(v, dtype=torch.float32)) for v in (low, high, kl))
    l, A, d = lp.double().requires_grad_(True), adv.double(), lp.double() - old.double()
    r = (l - old.double()).exp()
    t = -torch.minimum(r * A, r.clamp(1 - low, 1 + high) * A)
    (dt,) = torch.autograd.grad(t.sum(), [l])
    r, t = r.detach(), t.detach()
    cut = ((A > 0) & (r > 1 + high)) | ((A < 0) & (r < 1 - low))
    q = ref.double() - lp.double()
    one = torch.special.expm1(q)
    small = q.square() / 2 * (1 + q / 3 * (1 + q / 4 * (1 + q / 5)))             # its next term is below 1e-14 of it
    line = torch.where(q.abs() < 1e-3, small, one - q)
    e_t = torch.where(cut, 3.0, 7 + d.abs()) * t.abs() * U
    far = q.exp() * (4 + q.abs().nan_to_num(posinf=0.0)) + one.abs()
    e_one = torch.where(q.abs() < 1, q.abs() + 6 * line + one.abs(), far) * U
    e_line = torch.where(q.abs() < 1, 6 * line + q.abs() * one.abs(), far + line) * U
    sums = torch.stack([t.mean(), line.mean(), cut.double().mean(), torch.tensor(float(lp.numel()), dtype=torch.float64)])
    tols = torch.stack([e_t.mean(), e_line.mean(), sums[2] * 0, sums[3] * 0]) + 1.01 * U * sums.abs()
    e_dl = (torch.where(cut, 0.0, e_t) + kl * e_one + 4 * U * (dt.abs() + 2 * kl * one.abs())) / lp.numel()
    loss = sums[0] + kl * sums[1]
    return loss, sums, (dt - kl * one) / lp.numel(), (tols[0] + kl * tols[1] + 1.01 * U * loss.abs(), tols, e_dl)


def check_terms(lp, old, adv, ref, kl, dev):
    a = lp.to(dev).requires_grad_(True)
    loss, stats = ag.policy_loss(a, old.to(dev), adv.to(dev), ref_log_prob=ref.to(dev), kl_coef=kl, clip_high=0.28)
    (dl,) = torch.autograd.grad(loss, [a])
    w_loss, w_stats, w_dl, tols = policy_formula(lp, old, adv, ref, kl)
    w_stats[w_stats > torch.finfo(torch.float32).max] = math.inf
    close(loss, w_loss, tols[0], "loss")
    close(stats, w_stats, tols[1], "stats")
    close(dl, w_dl, tols[2], "gradient")


def test_policy_loss_terms(dev):
    M = 4097
    lp, old, ref = ratios(11, M)
    check_terms(lp, old, 1.0 + rnd(12, M).abs(), ref, 0.05, dev)
    check_terms(lp, old, rnd(13, M).sign(), lp + 2.0 * rnd(14, M), 0.5, dev)     # KL arguments of either side of 1


@pytest.mark.parametrize("q", [1e-6, -1e-3, 95.0, 100.0, -17.3, -20000.3, -1e8, -math.inf])
def test_policy_loss_of_a_far_reference(dev, q):
    """exp(q) past float32, whose share of the mean is not, and q so low that exp(q) - 1 is -1 whatever q is."""
    M = 100_003
    lp, old, ref = ratios(5, M)
    ref[70_000] = lp[70_000] + q
    check_terms(lp, old, 1.0 + rnd(6, M).abs(), ref, 0.04, dev)
    check_terms(lp[69_900:70_100], old[69_900:70_100], 1.0 + rnd(6, 200).abs(), ref[69_900:70_100], 1e-3, dev)


@pytest.mark.parametrize("d", [88.0, 90.0, 95.0, -100.0])
def test_policy_loss_of_a_far_old_model(dev, d):
    """A ratio past float32 that the clip leaves as it is (a negative advantage)."""
    M = 100_003
    lp, old, ref = ratios(5, M)
    adv = -1.0 - rnd(6, M).abs()
    old[70_000] = lp[70_000] - d
    check_terms(lp, old, adv, ref, 0.0, dev)
    check_terms(lp, old, adv, ref, 0.04, dev)


@pytest.mark.parametrize("V", [70, 300, 1000, 5001, 40003])
def test_log_prob_gradient_of_unlikely_classes(dev, V):
    """Every element of a float32 gradient to its last places, not only those that weigh in the row's sum.  One logit is 0 and
    the others are multiples of 1/8 from -60 to -20, so that differences from the largest are exact and the row's sum is 1 up to
    two roundings: what is left are the exponential (4 U), the sum (2 U), g over the sum (1 U), the product (1 U) and the class's
    own difference (1 U): 10 U with their products."""
    M = 5
    x = -(torch.randint(160, 481, (M, V), generator=torch.Generator().manual_seed(V)).float() / 8)
    x[:, V // 3] = 0.0
    x[M - 1] += 64.0                                     # about the largest logit, not about 0
    g = 1.0 + rnd(1, M).abs()
    c = torch.full((M,), V - 1)
    a = x.to(dev).requires_grad_(True)
    (dx,) = torch.autograd.grad(ag.class_log_prob(a, c.to(dev)), [a], g.to(dev))
    p = x.double().softmax(1)
    want = g.double()[:, None] * (torch.nn.functional.one_hot(c, V).double() - p)
    close(dx, want, 10 * U * want.abs(), "gradient")


def test_capture_looks_behind_casts_and_views(dev):
    """The leaf whose eager graph is alive may be behind a cast, a view or a layout copy that is recorded inside the capture."""
    x = rnd(1, 30, 64, dtype=torch.bfloat16).to(dev)
    w = (1 + 0.1 * rnd(2, 64)).to(dev).requires_grad_(True)
    emb = rnd(3, 40, 64).to(dev).requires_grad_(True)
    wide = rnd(4, 128).to(dev).requires_grad_(True)
    tok, off = torch.arange(30, device=dev), torch.tensor([0, 9, 64], device=dev)
    alive = [ag.layer_norm(x, w.bfloat16()), ag.token_embedding(emb.bfloat16(), tok), wide * 2]
    torch.cuda.synchronize()
    for call in (lambda: ag.layer_norm(x, w.bfloat16()), lambda: ag.token_embedding(emb.bfloat16(), tok),
                 lambda: ag.token_embedding(emb[:35], tok), lambda: ag.layer_norm(x.float(), wide[::2]),
                 lambda: ag.class_log_prob((x.float() * w).relu().exp(), tok), lambda: ag.policy_loss(w * 2, w.detach(), w.detach()),
                 lambda: ag.preference_loss(w * 2, w.detach(), off)):
        with pytest.raises(RuntimeError, match="same leaf tensor is alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive

    def step():
        y = ag.token_embedding(emb.bfloat16(), tok)
        y = ag.layer_norm(y + ag.token_embedding(emb[:35].bfloat16(), tok), w.bfloat16(), (wide[::2] * 1).bfloat16())
        loss, _ = ag.policy_loss(w * 2, w.detach(), w.detach(), offsets=None)
        pref, _ = ag.preference_loss(wide[::2] * 2, w.detach(), off)
        return [y.detach(), *torch.autograd.grad(y.float().square().mean() + loss + pref, [emb, w, wide])]

    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_losses_keep_no_workspace_for_the_backward(dev):
    """Between the passes a loss keeps its weights (4 bytes a sequence) and slopes (4 bytes an item), not what its sums needed (32 bytes a sequence).  The
    allocator leaves a rest of up to 1 MiB with a block of more than that; two are alive at most."""
    S, M = 1_000_000, 1_100_000
    off = (torch.arange(S + 1) * M // S).to(torch.int32).to(dev)
    lp = rnd(1, M).to(dev).requires_grad_(True)
    old, adv = rnd(2, M).to(dev), rnd(3, S).to(dev)
    for call, need in ((lambda: ag.policy_loss(lp, old, adv, offsets=off), 4 * (S + M)),
                       (lambda: ag.preference_loss(lp, old, off), 4 * S + 4 * S)):        # and the rewards
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(dev)
        out = call()
        assert torch.cuda.memory_allocated(dev) - before <= need + 2 * 2 ** 20 + 8192
        torch.autograd.grad(out[0], [lp])
        del out


@pytest.mark.parametrize("n, C", [(2, 1), (65, 1), (65, 33)])
def test_token_embedding_of_very_wide_rows(dev, n, C):
    """Rows of more tiles than a launch has in its second dimension: a gradient wherever there is a forward."""
    w = 65535 * 256 + 300
    W = (torch.arange(C, device=dev)[:, None] + torch.arange(w, device=dev)[None] % 50).float().requires_grad_(True)
    tok = torch.arange(n, device=dev) % C
    y = ag.token_embedding(W, tok)
    assert torch.equal(y[n - 1], W.detach()[tok[n - 1]])
    up = (torch.arange(w, device=dev) % 7).float().expand(n, w)                  # small whole numbers: exact sums
    (dW,) = torch.autograd.grad(y, [W], up)
    count = torch.bincount(tok, minlength=C).float()
    for c in range(C):
        assert torch.equal(dW[c], up[0] * count[c])


def test_log_prob_of_the_samplers_own_draws(dev):
    """class_log_prob of the log of BaseModel.posterior is the log-probability of an attribute as the sampler draws it: its own
    two posterior values (float32 products and sums of positive numbers, a few roundings each) normalised."""
    import numpy as np
    import graphmaker_amd as gm
    from graphmaker_amd import diffusion, ops
    n, F = 70, 9
    g = torch.Generator().manual_seed(3)
    marginal = torch.rand(F, generator=g) * 0.8 + 0.1
    marginal = torch.stack([1 - marginal, marginal], 1)
    trans = diffusion.MarginalTransition(dev, marginal.to(dev), torch.tensor([0.9, 0.1], device=dev), 2)
    alpha, abar_s, abar_t = np.float32(0.8), np.float32(0.5), np.float32(0.4)
    tab = torch.from_numpy(trans.table_X(alpha, abar_s, abar_t)).to(dev)
    logits = (2 * torch.randn(n, F, 2, generator=g)).to(dev).requires_grad_(True)
    x_t = torch.randint(0, 2, (n, F), generator=g, dtype=torch.uint8).to(dev)
    drawn, _, values = ops.attr_posterior_sample(logits.detach().reshape(n, 2 * F), x_t, tab, seed=4, step=1, want_debug=True)
    Z = torch.nn.functional.one_hot(x_t.t().long(), 2).float()                   # (F, n, 2)
    Q, Qs, Qt = (trans.get_Q_bar_X(float(a)) for a in (alpha, abar_s, abar_t))
    post = gm.ModelSync.posterior(None, Z, Q, Qs, Qt, logits.softmax(-1).transpose(0, 1)).transpose(0, 1)
    lp = ag.class_log_prob(post.log(), drawn.long())
    p = values.double().cpu()
    p = (p / p.sum(-1, keepdim=True)).gather(-1, drawn.long().cpu()[..., None])[..., 0]
    # float32: softmax, two tables, two products, a sum, the logarithm's argument: 32 U relative of a probability, and of the
    # logarithms as much of their size
    close(lp, p.log(), 32 * U * (1 + p.log().abs()), "log-probability of a draw")
    plain = ag.class_log_prob(logits, drawn.long())
    assert (plain.detach() - lp.detach()).abs().max() > 0.1                      # softmax(logits) is another distribution
    (dl,) = torch.autograd.grad(lp.sum(), [logits])
    assert dl.isfinite().all() and dl.any()


@pytest.mark.parametrize("M, N", [(1100, 16388), (600, 32772)])
def test_layer_norm_long_rows_in_turn(dev, M, N):
    """Rows that no workgroup holds, more of them than workgroups: the column sums go on from row to row."""
    check_norm((rnd(N, M, N) * (1 + torch.arange(M)[:, None] % 3) + 0.7), 1 + 0.3 * rnd(1, N), rnd(2, N), rnd(3, M, N), dev)


@pytest.mark.parametrize("dt", TYPES)
def test_rows_have_the_same_bits_at_any_alignment(dev, dt):
    t = DT[dt]
    for N in (3, 40, 512, 1000, 5001):
        M = 50
        base, gb = rnd(1, M, N + 9, dtype=t).to(dev), rnd(2, M, N + 9, dtype=t).to(dev)
        ga, be = (1 + 0.2 * rnd(3, N)).to(t).to(dev).requires_grad_(True), rnd(4, N, dtype=t).to(dev).requires_grad_(True)
        c = torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(3)).to(dev)
        g = rnd(4, M).to(dev)
        for at in (0, 1, 3, 8, 9):
            got = []
            for make in (lambda v: v, lambda v: v.contiguous()):
                x = make(base[:, at:at + N]).detach().requires_grad_(True)
                y = ag.layer_norm(x, ga, be)
                out = [y, *torch.autograd.grad(y, [x, ga, be], make(gb[:, at:at + N]))]
                lp = ag.class_log_prob(x, c)
                got.append(out + [lp, *torch.autograd.grad(lp, [x], g)])
            for k, (a, b) in enumerate(zip(*got)):
                assert torch.equal(a, b), (N, at, k)


def test_fine_tuning_gradients_against_differences_along_themselves(dev):
    """Every parameter's gradient of the whole chain, along its own direction (where the slope is its norm) and along a random
    one at right angles to it (where the slope is 0), against central differences of steps h and h/2 joined to fourth order.
    Their difference is 3/4 of what truncation leaves at h, and a fourth of it is allowed for what the joining leaves; the float32
    losses of about 1 are given 64 U of rounding each.  The tolerance has to be below a thousandth of the gradient's norm, so that
    the check has force.  The clip is opened: no ratio may cross a
    border of its range."""
    from test_gpu_finetune import fine_tuning_setup
    p, batch = fine_tuning_setup(dev, torch.float32)
    mask = batch["classes"] != -100

    def f(q):
        h = ag.layer_norm(ag.token_embedding(q["emb"], batch["tokens"], scale=4.0, padding_idx=0), q["gamma"], q["beta"])
        lp = ag.class_log_prob(ag.linear(h, q["W"], q["b"]), batch["classes"])
        a, _ = ag.policy_loss(lp, batch["old"], batch["adv"], offsets=batch["offsets"], mask=mask, ref_log_prob=batch["ref"], clip_low=1.0,
                              clip_high=100.0, kl_coef=0.05, reduction="sequence")
        b, _ = ag.preference_loss(lp, batch["ref"], batch["offsets"], mask=mask, beta=0.3)
        return a + b

    grads = dict(zip(p, torch.autograd.grad(f(p), list(p.values()))))
    for name, t in p.items():
        g = grads[name].double()
        along = g / g.norm()
        across = torch.randn(t.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64).to(dev)
        if name == "emb":
            across[0] = 0.0                              # the padding row: used, and without a gradient by definition
        across -= (across * along).sum() * along
        across /= across.norm()
        for v in (along, across):
            def quotient(step):
                with torch.no_grad():
                    up, down = (float(f({**p, name: (t.double() + s * v).float()}).double()) for s in (step, -step))
                return (up - down) / (2 * step)
            h = 1e-2
            wide, near = quotient(h), quotient(h / 2)
            got, want = (4 * near - wide) / 3, float((g * v).sum())
            # (4 (2 E) / h + (2 E) / (2 h)) / 3 with E = 64 U
            tol = abs(wide - near) / 4 + 3 * 64 * U / h
            assert tol < 1e-3 * float(g.norm()) and abs(got - want) <= tol, (name, got, want, tol)


def hooked_step(dev, dtype, strided):
    """Every operator's gradient, of inputs that are rows of wider tensors or packed."""
    def put(seed, *shape, dtype=torch.float32):
        t = rnd(seed, *shape[:-1], 2 * shape[-1] + 3, dtype=dtype).to(dev)[..., 3:3 + shape[-1]]
        return (t if strided else t.contiguous()).detach().requires_grad_(True)
    n, C, w = 90, 30, 72
    x, emb, logits, narrow, lp = put(1, n, w, dtype=dtype), put(2, C, w, dtype=dtype), put(3, n, 5003, dtype=dtype), put(4, n, 2), put(5, 12, 9)
    gamma, beta = put(6, w), put(7, w)
    tok, cls = (torch.arange(n, device=dev) * 7 % C).int(), torch.arange(n, device=dev) % 2
    mask, off = rnd(8, 12, 9).to(dev) > 0, torch.tensor([0, 30, 100], device=dev, dtype=torch.int32)
    old, adv = lp.detach() + 0.1, rnd(9, 2).to(dev)
    out = ag.layer_norm(x, gamma, beta).float().square().sum() + ag.token_embedding(emb, tok).float().square().sum()
    out = out + ag.class_log_prob(logits, cls).square().sum() + ag.class_log_prob(narrow, cls).sum()
    out = out + ag.policy_loss(lp, old, adv, offsets=off, mask=mask)[0] + ag.preference_loss(lp, old, off, mask=mask)[0]
    return out, [x, gamma, beta, emb, logits, narrow, lp]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("strided", [False, True])
def test_saved_tensors_may_be_moved(dev, dt, strided):
    """Hooks on saved tensors hand them back with strides of their own: kept in host memory, or cloned."""
    out, leaves = hooked_step(dev, DT[dt], strided)
    want = torch.autograd.grad(out, leaves)
    packed = torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)
    other = torch.autograd.graph.saved_tensors_hooks(lambda t: t.expand(2, *t.shape).movedim(0, -1).contiguous()[..., 0], lambda t: t)
    for hooks in (packed, other, torch.autograd.graph.save_on_cpu(pin_memory=False), torch.autograd.graph.save_on_cpu(pin_memory=True)):
        with hooks:
            out, leaves = hooked_step(dev, DT[dt], strided)
        for a, b in zip(torch.autograd.grad(out, leaves), want):
            assert torch.equal(a, b)
    y = torch.utils.checkpoint.checkpoint(lambda: hooked_step(dev, DT[dt], strided)[0], use_reentrant=False)
    assert torch.isfinite(y)


def test_saved_tensors_of_another_kind_are_refused(dev):
    """What comes back with another type, size or place would be read as what it is not."""
    x, w = rnd(1, 40, 64).to(dev).requires_grad_(True), rnd(2, 64).to(dev).requires_grad_(True)
    tok, off = torch.arange(40, device=dev), torch.tensor([0, 9, 40], device=dev)
    flat = rnd(3, 40).to(dev).requires_grad_(True)
    ref = rnd(4, 40).to(dev)
    for change in (lambda t: t.bfloat16() if t.is_floating_point() else t.int(), lambda t: t[:-1], lambda t: t.cpu()):
        for call, leaf in ((lambda: ag.layer_norm(x, w), x), (lambda: ag.token_embedding(x, tok), x), (lambda: ag.class_log_prob(x, tok), x),
                           (lambda: ag.policy_loss(flat, ref, ref)[0], flat), (lambda: ag.preference_loss(flat, ref, off)[0], flat)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                y = call()
            with pytest.raises(RuntimeError, match="came back as"):
                torch.autograd.grad(y.sum(), [leaf])


def test_second_derivatives_are_refused_however_they_are_asked_for(dev):
    """Also where only one path is differentiated and a missing one would count as zero: a Hessian, a Jacobian-vector product by
    two backward passes, a gradient's derivative after the upstream gradient."""
    x, w = rnd(1, 6, 40).to(dev), rnd(2, 40).to(dev)
    flat, ref = rnd(3, 6).to(dev), rnd(4, 6).to(dev)
    tok, off = torch.arange(6, device=dev), torch.tensor([0, 2, 6], device=dev)
    calls = [(lambda a: ag.layer_norm(a, w).square().sum(), x), (lambda a: ag.layer_norm(a[:, ::2]).sum(), x), (lambda a: ag.layer_norm(x, a).square().sum(), w),
             (lambda a: ag.token_embedding(a, tok).square().sum(), x), (lambda a: ag.class_log_prob(a, tok).sum(), x),
             (lambda a: ag.class_log_prob(a[:, :2], tok % 2).sum(), x), (lambda a: ag.policy_loss(a, ref, ref)[0], flat),
             (lambda a: ag.preference_loss(a, ref, off)[0], flat)]
    F = torch.autograd.functional
    for f, at in calls:
        for ask in (lambda: F.hessian(f, at), lambda: F.jvp(f, at, torch.ones_like(at)), lambda: F.hvp(f, at, torch.ones_like(at)), lambda: F.vhp(f, at, torch.ones_like(at))):
            with pytest.raises(RuntimeError, match="no second derivative"):
                ask()
        a, up = at.clone().requires_grad_(True), torch.ones((), device=dev, requires_grad=True)
        (da,) = torch.autograd.grad(f(a), [a], up, create_graph=True)
        for of in (a, up):
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(da.sum(), [of], allow_unused=True, retain_graph=True)
        del da
    assert torch.equal(F.vjp(calls[0][0], x)[1], F.jacobian(calls[0][0], x))     # one backward pass is fine


@pytest.mark.parametrize("dt, V", [("f32", 2), ("f32", 3), ("bf16", 2), ("bf16", 7), ("f16", 3), ("f16", 7)])
def test_log_prob_of_a_nearly_certain_class(dev, dt, V):
    """A draw of a sparse graph is nearly certain: log-probabilities of -1e-3 to -1e-20, and the gradient 1 - p of the class itself,
    keep their own last places, not those of 1.  The logits are multiples of 1/8 below 48 (the largest of them exact in any type), so that differences are exact: 4 U of an exponential,
    U of each of up to 6 sums and of 1 + the rest, 3 U of the logarithm and its correction, 2 U of a quotient and a product."""
    M = 2000
    gen = torch.Generator().manual_seed(V)
    x = -(torch.randint(8, 360, (M, V), generator=gen).float() / 8)
    top = torch.randint(0, V, (M,), generator=gen)
    x[torch.arange(M), top] = 0.0
    x += (torch.arange(M) % 5 - 2)[:, None]
    x = x.to(DT[dt])
    c = torch.where(torch.arange(M) % 4 > 0, top, (top + 1) % V)
    g = 1.0 + rnd(1, M).abs()
    a = x.to(dev).requires_grad_(True)
    lp = ag.class_log_prob(a, c.to(dev))
    (dx,) = torch.autograd.grad(lp, [a], g.to(dev))
    t = x.double() - x.double().gather(1, top[:, None])
    others = torch.nn.functional.one_hot(top, V).double()
    rest = (t.exp() * (1 - others)).sum(1)
    want = t.gather(1, c[:, None])[:, 0] - rest.log1p()
    assert float(want.abs().min()) < 1e-12
    close(lp, want, 16 * U * want.abs(), "log-probability")
    own = torch.nn.functional.one_hot(c, V).double()
    e = t.exp()
    grad = g.double()[:, None] / (1 + rest)[:, None] * (own * ((1 - own) * e).sum(1, keepdim=True) - (1 - own) * e)
    close(dx, grad, 16 * U * grad.abs() + torch.finfo(DT[dt]).eps / 2 * 1.01 * grad.abs()
          + torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps, "gradient")


@pytest.mark.parametrize("share", [0.5, 0.25])
def test_policy_loss_where_gains_cancel(dev, share):
    """Clipped items against items of ratio 1 whose advantages make up for them, up to the places that float32 does not have: the
    borders are 1 - clip_low and 1 + clip_high of the float32 arguments, and what is left is right to one rounding."""
    M = 4000
    n = int(M * share)
    low, high = (float(torch.tensor(v)) for v in (0.2, 0.28))
    for sign, border in ((1.0, 1 + high), (-1.0, 1 - low)):
        old, adv = torch.zeros(M), torch.full((M,), sign)
        old[:n] = -sign                                  # ratio e with an advantage, 1 / e with a disadvantage: clipped
        adv[n:] = -sign * border * n / (M - n)           # ratio 1
        a = torch.zeros(M, device=dev, requires_grad=True)
        loss, stats = ag.policy_loss(a, old.to(dev), adv.to(dev), clip_high=0.28)
        want = -(n * sign * border + adv[n:].double().sum()) / M
        assert 0 < abs(float(want)) < 4 * U
        close(loss, want, 1.01 * U * abs(float(want)) + 2.0 ** -50, "loss")
        assert float(stats[2]) == share
