"""GPU tests of token_embedding, layer_norm, class_log_prob, policy_loss and preference_loss against their definitions in
float64 on the CPU, from the same (rounded) inputs.

Tolerances count roundings.  u = 2^-24 is half a step of float32, ut half a step of the stored type.  A float32 sum of k
terms in any order is off by at most k u sum|terms|; the row kernels add a lane's share of a row one by one and join lanes
and waves pairwise, so D(N) = ceil(N / 64) + 16 bounds the additions any one term goes through.
"""
import math

import pytest
import torch

from graphmaker_amd import autograd as ag

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPES = ["f32", "bf16", "f16"]


def ut(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the distance of neighbouring values below the smallest normal one."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def D(n):
    return math.ceil(n / 64) + 16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return torch.device("cuda:0")


def close(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        t = tol[tuple(at)].item() if torch.is_tensor(tol) and tol.dim() == got.dim() else tol
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {at}: {got[tuple(at)].item()!r} for "
                             f"{want[tuple(at)].item()!r}, tolerance {t}")


def rnd(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------ token_embedding
def embedding_reference(weight, tokens, g, scale, padding):
    """(y, dW, sum of |terms| of dW, terms) in float64; a token outside the table: NaN row, no gradient."""
    C, w = weight.shape
    W, t = weight.double(), tokens.reshape(-1).long()
    ok = (t >= 0) & (t < C)
    y = torch.full((t.numel(), w), math.nan, dtype=torch.float64)
    y[ok] = W[t[ok]] * scale
    keep = ok if padding is None else ok & (t != padding % C)        # a negative padding_idx counts from the end
    gd = g.reshape(-1, w).double()[keep]
    dW = torch.zeros(C, w, dtype=torch.float64).index_add_(0, t[keep], gd) * scale
    size = torch.zeros(C, w, dtype=torch.float64).index_add_(0, t[keep], gd.abs()) * abs(scale)
    count = torch.bincount(t[keep], minlength=C)[:, None].double()
    return y.reshape(tokens.shape + (w,)), dW, size, count


def check_embedding(weight, tokens, scale, padding, dev, seed=1):
    dt = weight.dtype
    g = rnd(seed, *tokens.shape, weight.shape[1], dtype=dt)
    W = weight.to(dev).requires_grad_(True)
    y = ag.token_embedding(W, tokens.to(dev), scale=scale, padding_idx=padding)
    (dW,) = torch.autograd.grad(y, [W], g.to(dev))
    wy, wdW, size, count = embedding_reference(weight, tokens, g, scale, padding)
    close(y, wy, (ut(dt) + 2 * U) * wy.abs().nan_to_num() + tiny(dt), "embedding")
    close(dW, wdW, (count + 2) * U * size + ut(dt) * wdW.abs() * 1.01 + tiny(dt), "embedding gradient")
    with torch.no_grad():
        assert torch.equal(ag.token_embedding(W, tokens.to(dev), scale=scale, padding_idx=padding).nan_to_num(), y.nan_to_num())
    return dW


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n, C, w", [(1, 1, 1), (1, 300, 8), (7, 5, 3), (64, 2, 64), (65, 511, 66), (513, 512, 33), (2049, 513, 128),
                                     (1000, 100003, 16), (5000, 10, 65), (4097, 262145, 8), (100, 7, 1030), (8193, 33, 40),
                                     (150001, 200000, 3), (300001, 1000, 2), (70001, 32, 9)])
def test_token_embedding(dev, dt, n, C, w):
    g = torch.Generator().manual_seed(n + C + w)
    tokens = (torch.rand(n, generator=g) ** 3 * C).long().clamp(max=C - 1)       # low rows often, most never
    check_embedding(rnd(3, C, w, dtype=DT[dt]), tokens, 1.7, None, dev)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_token_embedding_shapes_padding_and_bad_tokens(dev, index):
    C, w = 37, 24
    W = rnd(5, C, w)
    t = torch.randint(0, C, (6, 11), generator=torch.Generator().manual_seed(2))
    t[:, 8:] = 4
    check_embedding(W, t.to(index), 0.5, 4, dev)
    a = check_embedding(W, t.to(index), 1.0, C - 1, dev)
    b = check_embedding(W, t.to(index), 1.0, -1, dev)                            # counted from the end
    assert torch.equal(a, b)
    t[0, 0], t[1, 1], t[2, 2] = -1, C, 2 ** 31 - 1
    check_embedding(W, t.to(index), 1.0, None, dev)
    t[:] = -7
    check_embedding(W, t.to(index), 1.0, None, dev)                              # no token adds to any row
    if index == torch.int64:
        t[3, 3], t[4, 4] = 2 ** 32 + 3, -(2 ** 40)                               # would be in range if cut to 32 bits
        check_embedding(W, t, 1.0, None, dev)


@pytest.mark.parametrize("n, C", [(6000, 3), (40000, 1), (9000, 70000), (30011, 600)])
def test_token_embedding_hot_rows(dev, n, C):
    """Rows with thousands of tokens, alone or among rows with one, with runs that end at borders of any power of two."""
    t = torch.arange(n) % C
    t[: n // 2] = C // 2
    p = torch.randperm(n, generator=torch.Generator().manual_seed(4))
    check_embedding(rnd(6, C, 16), t[p], 1.0, None, dev)
    check_embedding(rnd(6, C, 16), t, 1.0, None, dev)
    check_embedding(rnd(6, C, 16), torch.full((n,), C // 2), 1.0, None, dev)
    check_embedding(rnd(6, C, 16), torch.full((n,), C // 2), 1.0, C // 2, dev)   # all padding


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n, C, w", [(2, 82, 559), (63, 40, 3), (64, 1000, 40), (64, 3, 1030), (65, 1000, 40), (16385, 5000, 5), (300001, 90000, 1)])
def test_token_embedding_bad_tokens_and_padding(dev, dt, n, C, w):
    """Around the borders of the gradient's forms: the same token often, tokens outside the table on either side, padding."""
    t = torch.randint(-2, C + 2, (n,), generator=torch.Generator().manual_seed(n))
    t[::3] = C // 3
    check_embedding(rnd(9, C, w, dtype=DT[dt]), t, 0.7, C // 2, dev)
    check_embedding(rnd(9, C, w, dtype=DT[dt]), t.to(torch.int32), 1.0, C // 3, dev)


def test_token_embedding_is_reproducible_and_strided(dev):
    C, w, n = 5000, 40, 9001
    t = (torch.rand(n, generator=torch.Generator().manual_seed(1)) ** 4 * C).long().to(dev)
    big = rnd(7, C, 2 * w + 3).to(dev)
    g = rnd(8, n, 3 * w).to(dev)
    view, gview = big[:, 3:3 + w].detach().requires_grad_(True), g[:, w:2 * w]
    y = ag.token_embedding(view, t, scale=2.0)
    (dv,) = torch.autograd.grad(y, [view], gview)
    whole = big[:, 3:3 + w].contiguous().requires_grad_(True)
    z = ag.token_embedding(whole, t, scale=2.0)
    (dw,) = torch.autograd.grad(z, [whole], gview.contiguous())
    assert torch.equal(y, z) and torch.equal(dv, dw)
    for _ in range(3):
        z = ag.token_embedding(whole, t, scale=2.0)
        assert torch.equal(torch.autograd.grad(z, [whole], gview)[0], dw)
    column = big.t()[:, :w].detach().requires_grad_(True)                        # column-major weight
    y = ag.token_embedding(column, t % column.shape[0])
    assert torch.equal(y, column.detach()[t % column.shape[0]])
    (dc,) = torch.autograd.grad(y.sum(), [column])                               # an expanded upstream gradient
    want = torch.bincount(t % column.shape[0], minlength=column.shape[0]).float()
    assert torch.equal(dc, want[:, None].expand(-1, w))                          # small whole numbers: exact
    empty = ag.token_embedding(whole, t[:0])
    assert empty.shape == (0, w) and torch.equal(torch.autograd.grad(empty.sum(), [whole])[0], torch.zeros_like(whole))


# ------------------------------------------------------------------ layer_norm
def check_norm(x, gamma, beta, g, dev, eps=1e-5):
    dt, N = x.dtype, x.shape[-1]
    args = [t.to(dev).requires_grad_(True) if t is not None else None for t in (x, gamma, beta)]
    y = ag.layer_norm(*args, eps=eps)
    live = [t for t in args if t is not None]
    grads = list(torch.autograd.grad(y, live, g.to(dev)))
    X, G = x.double().reshape(-1, N), g.double().reshape(-1, N)
    ga = gamma.double() if gamma is not None else torch.ones(N, dtype=torch.float64)
    be = beta.double() if beta is not None else torch.zeros(N, dtype=torch.float64)
    mu = X.mean(1, keepdim=True)
    r = 1.0 / ((X - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (X - mu) * r
    # xh: the mean is off by D u mean|x|, the variance by a share of (D + 4) u and twice the mean's error over the spread
    d = D(N)
    e_mu = d * U * X.abs().mean(1, keepdim=True) * r
    e_xh = e_mu + U * (X * r).abs() + xh.abs() * ((d + 8) * U + e_mu * e_mu)
    want = xh * ga + be
    close(y.reshape(-1, N), want, ga.abs() * e_xh + 4 * U * ((xh * ga).abs() + be.abs()) + ut(dt) * want.abs() * 1.01 + tiny(dt), "norm")
    gg = G * ga
    s1, s2 = gg.mean(1, keepdim=True), (gg * xh).mean(1, keepdim=True)
    dx = r * (gg - s1 - xh * s2)
    e_s1 = d * U * gg.abs().mean(1, keepdim=True)
    e_s2 = (d + 2) * U * (gg * xh).abs().mean(1, keepdim=True) + (gg.abs() * e_xh).mean(1, keepdim=True)
    e_dx = r * (e_s1 + xh.abs() * e_s2 + e_xh * s2.abs() + 4 * U * (gg.abs() + s1.abs() + (xh * s2).abs()))
    e_dx = e_dx + dx.abs() * ((d + 8) * U + e_mu * e_mu) + ut(dt) * dx.abs() * 1.01 + tiny(dt)
    close(grads.pop(0).reshape(-1, N), dx, e_dx, "norm dx")
    m = X.shape[0] + 16
    if gamma is not None:
        wt = gamma.dtype
        w = (G * xh).sum(0)
        close(grads.pop(0), w, (G.abs() * e_xh).sum(0) + m * U * (G * xh).abs().sum(0) + ut(wt) * w.abs() * 1.01 + tiny(wt), "norm dgamma")
    if beta is not None:
        wt = beta.dtype
        close(grads.pop(0), G.sum(0), m * U * G.abs().sum(0) + ut(wt) * G.sum(0).abs() * 1.01 + tiny(wt), "norm dbeta")
    with torch.no_grad():
        assert torch.equal(ag.layer_norm(*args, eps=eps), y)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M, N", [(1, 1), (1, 2), (3, 7), (5, 64), (4, 65), (130, 96), (67, 512), (1, 1000), (9, 1023), (64, 1024),
                                  (3, 2049), (2, 4096), (33, 5000), (7, 8192), (5, 16384), (2, 20001), (1, 70000), (700, 24),
                                  (5000, 96), (1300, 2056), (300, 16400), (20, 700), (20, 1500), (2, 40000), (9000, 40)])
def test_layer_norm(dev, dt, M, N):
    t = DT[dt]
    x = (rnd(N, M, N) * (1 + torch.arange(M)[:, None] % 3) + 0.7).to(t)
    check_norm(x, (1 + 0.3 * rnd(1, N)).to(t), rnd(2, N, dtype=t), rnd(3, M, N, dtype=t), dev)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("M, N", [(5, 96), (40, 1024), (3, 9001)])
def test_layer_norm_with_float_weights(dev, dt, M, N):
    check_norm(rnd(1, M, N, dtype=DT[dt]), 1 + 0.3 * rnd(2, N), rnd(3, N), rnd(4, M, N, dtype=DT[dt]), dev)


def test_layer_norm_absent_weights_shapes_offsets(dev):
    x, g = rnd(1, 2, 3, 5, 40), rnd(2, 2, 3, 5, 40)
    check_norm(x, None, None, g, dev)
    check_norm(x, rnd(3, 40), None, g, dev)
    check_norm(x, None, rnd(4, 40), g, dev)
    check_norm(1000.0 + x, rnd(3, 40), rnd(4, 40), g, dev)                       # a mean far above the spread
    check_norm(torch.full((4, 40), 3.25), rnd(3, 40), rnd(4, 40), rnd(5, 4, 40), dev)        # no spread at all
    y = ag.layer_norm(torch.empty(0, 40, device=dev))
    assert y.shape == (0, 40)
    w = rnd(3, 40).to(dev).requires_grad_(True)
    y = ag.layer_norm(torch.empty(0, 40, device=dev), w)
    assert torch.equal(torch.autograd.grad(y.sum(), [w])[0], torch.zeros(40, device=dev))


@pytest.mark.parametrize("dt", TYPES)
def test_layer_norm_strides_and_alignment(dev, dt):
    """Rows further apart than their width, starting anywhere, columns out of order: the bits of the packed copy."""
    t = DT[dt]
    base, gb = rnd(1, 50, 700, dtype=t).to(dev), rnd(2, 50, 700, dtype=t).to(dev)
    ga, be = (1 + 0.2 * rnd(3, 512)).to(t).to(dev).requires_grad_(True), rnd(4, 512, dtype=t).to(dev).requires_grad_(True)
    for at in (0, 1, 3, 8):
        got, want = [], []
        for out, make in ((got, lambda v: v), (want, lambda v: v.contiguous())):
            x = make(base[:, at:at + 512]).detach().requires_grad_(True)
            y = ag.layer_norm(x, ga, be)
            out += [y, *torch.autograd.grad(y, [x, ga, be], make(gb[:, at:at + 512]))]
        for a, b in zip(got, want):
            close(a, b.detach().cpu(), b.detach().cpu().double().abs() * (2 * ut(t) + 64 * U) + 1e-5, f"offset {at}")
    x = base.t()
    assert torch.equal(ag.layer_norm(x), ag.layer_norm(x.contiguous()))
    x = base[0].expand(6, 700)
    assert torch.equal(ag.layer_norm(x)[5], ag.layer_norm(base[0]))
    x = base[::3]
    assert torch.equal(ag.layer_norm(x), ag.layer_norm(x.contiguous()))


def test_layer_norm_nan_stays_in_its_row(dev):
    x, g = rnd(1, 9, 300), rnd(2, 9, 300)
    x[4, 7], x[6, 0] = math.nan, math.inf
    a = x.to(dev).requires_grad_(True)
    y = ag.layer_norm(a)
    (dx,) = torch.autograd.grad(y, [a], g.to(dev))
    bad = torch.tensor([4, 6])
    rest = torch.tensor([i for i in range(9) if i not in (4, 6)])
    assert y[bad.to(dev)].isnan().any(1).all() and y[rest.to(dev)].isfinite().all() and dx[rest.to(dev)].isfinite().all()


def test_wide_update_block_trains(dev):
    """Linear -> ReLU -> LayerNorm wider than 1024 columns, forward and gradients against float64."""
    M, K, N = 70, 48, 1500
    x, W, b = rnd(1, M, K), rnd(2, N, K) / K ** 0.5, 0.1 * rnd(3, N)
    gamma, beta, g = 1 + 0.1 * rnd(4, N), 0.1 * rnd(5, N), rnd(6, M, N)
    cpu = [t.double().requires_grad_(True) for t in (x, W, b, gamma, beta)]
    a = torch.relu(cpu[0] @ cpu[1].t() + cpu[2])
    xc = a - a.mean(1, keepdim=True)
    ref = xc / (xc.square().mean(1, keepdim=True) + 1e-5).sqrt() * cpu[3] + cpu[4]
    want = torch.autograd.grad(ref, cpu, g.double())
    gpu = [t.to(dev).requires_grad_(True) for t in (x, W, b, gamma, beta)]
    out = ag.update_block(*gpu, 1e-5)
    got = torch.autograd.grad(out, gpu, g.to(dev))
    close(out, ref.detach(), 2e-5 + 1e-5 * ref.detach().abs(), "wide update block")
    for what, p, q in zip(("dx", "dW", "db", "dgamma", "dbeta"), got, want):     # sums of up to 1500 products of O(1)
        close(p, q, 3e-5 * q.abs().max() + 1e-4 * q.abs(), f"wide update block {what}")


# ------------------------------------------------------------------ class_log_prob
def check_log_prob(x, c, g, dev, ignore=-100, index=torch.int64):
    dt, V = x.dtype, x.shape[-1]
    a = x.to(dev).requires_grad_(True)
    lp = ag.class_log_prob(a, c.to(index).to(dev), ignore_index=ignore)
    (dx,) = torch.autograd.grad(lp, [a], g.to(dev))
    X, cc, G = x.double().reshape(-1, V), c.reshape(-1), g.double().reshape(-1)
    out = torch.zeros(X.shape[0], dtype=torch.float64)
    dX = torch.zeros_like(X)
    tol, dtol = torch.zeros_like(out), torch.zeros_like(X)
    d = D(V)
    for i in range(X.shape[0]):
        if cc[i] == ignore:
            continue
        if not 0 <= cc[i] < V:
            out[i] = math.nan
            dX[i] = math.nan if G[i] != 0 else 0.0
            continue
        t = X[i] - X[i].max()
        ls = t.exp().sum().log()
        p = (t - ls).exp()
        out[i] = t[cc[i]] - ls
        # each exponential: 4 u and u |t| from the rounded difference; the sum D u; the logarithm 2 u of itself
        mean_t = (p * t.abs().nan_to_num(posinf=0.0)).sum()
        tol[i] = (d + 8) * U + U * mean_t + 4 * U * (ls.abs() + t[cc[i]].abs().nan_to_num(posinf=0.0)) + U * out[i].abs().nan_to_num(posinf=0.0)
        one = torch.zeros(V, dtype=torch.float64)
        one[cc[i]] = 1.0
        dX[i] = G[i] * (one - p) if G[i] != 0 else 0.0
        e_p = p * (U * (d + 16) + U * mean_t + 3 * U * (t.abs().nan_to_num(posinf=0.0) + ls.abs()))
        dtol[i] = G[i].abs() * (e_p + 2 * U * (one + p)) + ut(dt) * dX[i].abs() * 1.01 + tiny(dt) + 1e-38
    close(lp.reshape(-1), out, tol, f"log prob {tuple(x.shape)}")
    close(dx.reshape(-1, V), dX, dtol, f"log prob gradient {tuple(x.shape)}")
    with torch.no_grad():
        assert torch.equal(ag.class_log_prob(a, c.to(index).to(dev), ignore_index=ignore).nan_to_num(), lp.nan_to_num())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M, V", [(1, 1), (1, 2), (257, 2), (300, 3), (65, 5), (64, 10), (33, 16), (31, 17), (9, 33), (70, 64), (5, 65),
                                  (17, 100), (6, 257), (4, 512), (3, 1000), (9, 1025), (2, 4096), (5, 5003), (1, 9001), (3, 33001),
                                  (1, 131075), (40, 8192), (7, 1600), (5, 2400)])
def test_class_log_prob(dev, dt, M, V):
    g = torch.Generator().manual_seed(M * 7 + V)
    x = (2.0 * torch.randn(M, V, generator=g)).to(DT[dt])
    c = torch.randint(0, V, (M,), generator=g)
    if M > 4:
        c[2] = -100
    check_log_prob(x, c, torch.randn(M, generator=g), dev, index=torch.int32 if V % 2 else torch.int64)


@pytest.mark.parametrize("V", [2, 3, 10, 70, 700, 6000, 40000])
def test_class_log_prob_special_rows(dev, V):
    """Banned classes, NaN and infinities in rows that are ignored, classes outside the table, zero upstream gradients."""
    M = 12
    x = rnd(V, M, V)
    c = torch.randint(0, V, (M,), generator=torch.Generator().manual_seed(1))
    g = rnd(2, M)
    x[0], c[0] = math.nan, -100                          # ignored: not read
    x[1], c[1] = math.inf, -100
    x[2, 1:] = -math.inf                                 # one class left
    c[2] = 0
    x[3, 0], c[3] = -math.inf, 0                         # the class itself is banned
    c[4], c[5] = V, -1
    c[6], g[6] = V, 0.0
    g[7] = 0.0
    x[8] += 80.0                                         # exponentials about the largest logit, not about 0
    x[9] = torch.finfo(torch.float32).min                # the lowest value everywhere: uniform
    x[10] -= 1e4
    x[11, V // 2] = 60.0                                 # a certain class
    c[11] = V // 2
    check_log_prob(x, c, g, dev)
    lowest = x[8:9].to(torch.bfloat16)
    lowest[0, V // 2] = torch.finfo(torch.bfloat16).min
    check_log_prob(lowest, c[8:9], g[8:9], dev)
    y = x.clone()
    y[:, V - 1], c[:] = math.nan, 0
    a = y.to(dev).requires_grad_(True)
    lp = ag.class_log_prob(a, c.to(dev))
    assert lp.isnan().all()                              # a NaN that is not ignored shows
    assert ag.class_log_prob(torch.full((2, V), -math.inf, device=dev), c[:2].to(dev)).isnan().all()
    ones = torch.full((2, V), 1.0, device=dev)
    ones[:, 0] = math.inf
    assert ag.class_log_prob(ones, c[:2].to(dev)).isnan().all()
    check_log_prob(rnd(1, M, V), torch.full((M,), V - 1), g, dev, ignore=V - 1)          # an ignore_index inside the table
    check_log_prob(rnd(1, M, V), torch.full((M,), V - 1), g, dev, ignore=0)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2, 7, 600, 5001])
def test_class_log_prob_strides_shapes(dev, dt, V):
    t = DT[dt]
    base = rnd(1, 40, V + 9, dtype=t).to(dev)
    c = torch.randint(0, V, (40,), generator=torch.Generator().manual_seed(3)).to(dev)
    g = rnd(4, 40).to(dev)
    for at in (0, 1, 2, 4, 9):
        x, p = base[:, at:at + V].detach().requires_grad_(True), base[:, at:at + V].contiguous().requires_grad_(True)
        a, b = ag.class_log_prob(x, c), ag.class_log_prob(p, c)
        close(a, b.detach().cpu(), 64 * U * (1 + b.detach().cpu().double().abs()), f"offset {at}")
        da, db = torch.autograd.grad(a, [x], g)[0], torch.autograd.grad(b, [p], g)[0]
        close(da, db.detach().cpu(), db.detach().cpu().double().abs() * 2 * ut(t) + 256 * U * g.detach().cpu().double().abs()[:, None], f"offset {at}")
    x = base.t()[:V].t()
    assert torch.equal(ag.class_log_prob(x, c), ag.class_log_prob(x.contiguous(), c))
    four = rnd(5, 2, 3, 4, V, dtype=t).to(dev).requires_grad_(True)
    cc = torch.randint(0, V, (2, 3, 4), generator=torch.Generator().manual_seed(3)).to(dev)
    lp = ag.class_log_prob(four, cc)
    assert lp.shape == (2, 3, 4) and torch.autograd.grad(lp.sum(), [four])[0].shape == four.shape
    assert ag.class_log_prob(four[:0], cc[:0]).shape == (0, 3, 4)
    e = four[:0].detach().requires_grad_(True)
    assert torch.autograd.grad(ag.class_log_prob(e, cc[:0]).sum(), [e])[0].shape == e.shape


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V, times", [(2, 70000), (3, 9000), (7, 9000), (10, 9000), (100, 2000), (601, 600), (2049, 60), (5001, 60)])
def test_a_row_does_not_depend_on_the_rows_around_it(dev, dt, V, times):
    """The same 70 rows at other places of a larger batch, at other alignments and in other workgroups: the same bits, of the
    log-probabilities and their gradients, and of layer_norm's rows."""
    x = rnd(V, 70, V, dtype=DT[dt]).to(dev)
    c = torch.randint(0, V, (70,), generator=torch.Generator().manual_seed(1)).to(dev)
    g = rnd(2, 70).to(dev)
    shift = 13                                           # the batch starts with the last rows
    big = torch.cat([x[-shift:], x.repeat(times, 1)]).requires_grad_(True)
    lp = ag.class_log_prob(big, torch.cat([c[-shift:], c.repeat(times)]))
    (dx,) = torch.autograd.grad(lp, [big], torch.cat([g[-shift:], g.repeat(times)]))
    first, grad = lp[:70], dx[:70]
    for k in (1, times // 2, times - 1):
        assert torch.equal(lp[70 * k:70 * k + 70], first) and torch.equal(dx[70 * k:70 * k + 70], grad)
    y = ag.layer_norm(big.detach())
    few = ag.layer_norm(big.detach()[:70])
    assert torch.equal(y[:70], few) and torch.equal(y[70 * (times - 1):70 * times], few)


def test_second_derivatives_are_refused(dev):
    """create_graph is allowed; differentiating the gradient is an error, not silent zeros."""
    x = rnd(1, 6, 40).to(dev).requires_grad_(True)
    y = ag.layer_norm(x)
    (dx,) = torch.autograd.grad(y.square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.sum().backward()
    lp = ag.class_log_prob(x, torch.zeros(6, dtype=torch.int64, device=dev))
    (dx,) = torch.autograd.grad(lp.square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.sum().backward()


def test_tensors_on_different_devices_are_refused(dev):
    W, x = torch.zeros(4, 8, device=dev), torch.zeros(6, device=dev)
    for call in (lambda: ag.token_embedding(W, torch.zeros(3, dtype=torch.int64)), lambda: ag.layer_norm(W, torch.ones(8)),
                 lambda: ag.class_log_prob(W, torch.zeros(4, dtype=torch.int64)), lambda: ag.policy_loss(x, torch.zeros(6), x),
                 lambda: ag.policy_loss(x, x, x, mask=torch.ones(6, dtype=torch.bool)),
                 lambda: ag.preference_loss(x, x, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="expected cuda"):
            call()


def test_class_log_prob_equals_the_two_class_cross_entropy(dev):
    """Beside the framework's own loss of the same logits: mean of -log_prob = softmax_ce2."""
    x, y = rnd(1, 5000, 2).to(dev), torch.randint(0, 2, (5000,), generator=torch.Generator().manual_seed(2)).to(dev)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    one = -ag.class_log_prob(a, y).mean()
    two = ag.softmax_ce2(b, y.to(torch.uint8))
    one.backward()
    two.backward()
    one, two = float(one.detach()), float(two.detach())
    assert abs(one - two) <= 1e-5 * abs(two)                # the mean of 5000 float32 terms
    assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=1e-9)


# ------------------------------------------------------------------ losses
def sequences(offsets, M):
    """Sequence of each item (-1: in none)."""
    seq = torch.full((M,), -1)
    for s in range(len(offsets) - 1):
        seq[offsets[s]:offsets[s + 1]] = s
    return seq


def policy_reference(lp, old, adv, ref, mask, offsets, low, high, kl, reduction):
    """(loss, stats, dlp and tolerances) in float64."""
    M = lp.numel()
    seq = sequences(offsets, M) if offsets is not None else torch.zeros(M, dtype=torch.long)
    live = (seq >= 0) & (mask.bool() if mask is not None else True)
    A = torch.zeros(M, dtype=torch.float64)
    A[live] = adv.double()[seq[live]] if offsets is not None else adv.double()[live]
    S = len(offsets) - 1 if offsets is not None else 1
    count = torch.bincount(seq[live], minlength=S).double()
    wt = torch.zeros(M, dtype=torch.float64)
    if live.any():
        wt[live] = 1.0 / live.sum() if reduction == "token" else 1.0 / (count[seq[live]] * (count > 0).sum())
    z = torch.zeros(M, dtype=torch.float64)
    l, o = torch.where(live, lp.double(), z), torch.where(live, old.double(), z)
    q = torch.where(live, ref.double(), z) - l if ref is not None else z
    r = (l - o).exp()
    cut = ((A > 0) & (r > 1 + high)) | ((A < 0) & (r < 1 - low))
    t = -torch.minimum(r * A, r.clamp(1 - low, 1 + high) * A)
    k = torch.special.expm1(q) - q
    loss = (wt * (t + kl * k)).sum()
    stats = torch.stack([(wt * t).sum(), (wt * k).sum(), (wt * cut).sum(), live.sum().double()])
    dl = wt * (torch.where(cut, 0.0, -A * r) - kl * torch.special.expm1(q))
    e_t = torch.where(r > 0, (A * r).abs() * U * (8 + (l - o).abs()), 0.0)       # exp(-inf) = 0 has no error
    e_k = 12 * U * k + U * q.abs() * torch.special.expm1(q).abs() + torch.where(q.abs() >= 1, 4 * U * (q.exp() + q.abs()), 0.0)
    e_dl = e_t + kl * (4 * U * torch.special.expm1(q).abs() + e_k + U * q.abs() * (1 + q.exp()))
    tols = ((wt * (e_t + kl * e_k)).sum() + 4 * U * loss.abs(), torch.stack(
        [(wt * e_t).sum() + 2 * U * stats[0].abs(), (wt * e_k).sum() + 2 * U * stats[1], 2 * U * stats[2], U * stats[3]]),
        wt * e_dl + 4 * U * (wt * (A * r).abs() + wt * kl * torch.special.expm1(q).abs()))
    return loss, stats, dl, tols


def check_policy(lp, old, adv, dev, ref=None, mask=None, offsets=None, kl=0.0, reduction="token", low=0.2, high=0.28, index=torch.int32):
    a = lp.to(dev).requires_grad_(True)
    put = lambda t: t.to(dev) if t is not None else None  # noqa: E731
    kw = dict(offsets=torch.tensor(offsets, dtype=index).to(dev) if offsets is not None else None, mask=put(mask), ref_log_prob=put(ref),
              clip_low=low, clip_high=high, kl_coef=kl, reduction=reduction)
    loss, stats = ag.policy_loss(a, old.to(dev), adv.to(dev), **kw)
    assert loss.shape == () and not stats.requires_grad
    (dl,) = torch.autograd.grad(3.0 * loss, [a])
    w_loss, w_stats, w_dl, tols = policy_reference(lp, old, adv, ref, mask, offsets, low, high, kl, reduction)
    close(loss, w_loss, tols[0], "policy loss")
    close(stats, w_stats, tols[1] + 1e-45, "policy stats")
    close(dl, 3.0 * w_dl, 3.0 * tols[2] + 8 * U * w_dl.abs() + 1e-44, "policy gradient")
    with torch.no_grad():
        again = ag.policy_loss(a, old.to(dev), adv.to(dev), **kw)
        assert torch.equal(again[0], loss) and torch.equal(again[1], stats)


def ratios(seed, M, low=0.2, high=0.28):
    """(log_prob, old, ref): log ratios of size 0.2, none within 1e-4 of a border of the clip range, where the gradient jumps."""
    lp = -rnd(seed, M).abs()
    d = 0.2 * rnd(seed + 1, M)
    for b in (math.log(1 - low), math.log(1 + high)):
        d = torch.where((d - b).abs() < 1e-4, d + 3e-4, d)
    return lp, lp - d, lp + 0.3 * rnd(seed + 2, M)


@pytest.mark.parametrize("M", [1, 2, 63, 64, 65, 255, 1023, 1024, 1025, 4097, 70001])
def test_policy_loss_per_item(dev, M):
    lp, old, ref = ratios(M, M)
    adv = rnd(9, M)
    mask = torch.rand(M, generator=torch.Generator().manual_seed(M)) < 0.6
    check_policy(lp, old, adv, dev)
    check_policy(lp, old, adv, dev, ref=ref, kl=0.05, mask=mask)
    check_policy(lp, old, adv, dev, ref=ref, mask=mask.to(torch.uint8))          # KL reported, not in the loss


def ragged(seed, S, M):
    """Borders of S sequences in M items: short, long and empty ones, first and last at the ends or not."""
    g = torch.Generator().manual_seed(seed)
    cuts = (torch.rand(S + 1, generator=g) ** 2 * M).long().sort().values
    if seed % 2:
        cuts[0], cuts[-1] = 0, M
    if S > 3:
        cuts[2] = cuts[1]
    return cuts.tolist()


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("S, M", [(1, 1), (1, 5000), (2, 3), (5, 1024), (7, 9000), (64, 3001), (65, 3001), (300, 20000), (500, 400), (3000, 6000),
                                  (20000, 60000), (17000, 900)])
def test_policy_loss_of_sequences(dev, reduction, S, M):
    lp, old, ref = ratios(S + M, M)
    mask = torch.rand(M, generator=torch.Generator().manual_seed(M)) < 0.6
    for k, (off, m) in enumerate([(ragged(2 * S, S, M), None), (ragged(2 * S + 1, S, M), mask)]):
        lp2, old2 = lp.clone(), old.clone()
        outside = sequences(off, M) < 0
        lp2[outside], old2[outside] = math.nan, math.inf                         # rows behind the last sequence hold anything
        check_policy(lp2, old2, rnd(3, S), dev, ref=ref, mask=m, offsets=off, kl=0.04, reduction=reduction,
                     index=torch.int64 if k else torch.int32)


def test_policy_loss_masked_values_and_empty_batches(dev):
    M = 700
    lp, old, ref = ratios(1, M)
    mask = torch.ones(M, dtype=torch.bool)
    mask[100:300] = False
    for t, v in ((lp, math.nan), (old, -math.inf), (ref, math.inf)):
        t[100:300] = v
    adv = rnd(2, M)
    adv[100:300] = math.nan
    for red, off, a in (("token", None, adv), ("sequence", [0, 100, 300, 700], rnd(3, 3)), ("token", [0, 100, 300, 700], rnd(3, 3))):
        check_policy(lp, old, a, dev, ref=ref, mask=mask, kl=0.1, offsets=off, reduction=red)
    none = torch.zeros(M, dtype=torch.bool)
    for red, off, a in (("token", None, adv), ("sequence", [0, 100, 300, 700], rnd(3, 3)), ("token", [9, 9, 9], rnd(3, 2)), ("sequence", [9, 9, 9], rnd(3, 2))):
        check_policy(lp, old, a, dev, ref=ref, mask=none if off is None or len(off) > 3 else None, kl=0.1, offsets=off, reduction=red)
    e = torch.empty(0, device=dev, requires_grad=True)
    loss, stats = ag.policy_loss(e, e.detach(), e.detach())
    assert float(loss) == 0.0 and torch.equal(stats, torch.zeros(4, device=dev))
    assert torch.autograd.grad(loss, [e])[0].shape == (0,)
    loss, _ = ag.policy_loss(e, e.detach(), rnd(1, 2).to(dev), offsets=torch.zeros(3, dtype=torch.int32, device=dev))
    assert float(loss) == 0.0


def test_policy_loss_extremes(dev):
    """Advantages of zero, banned draws (log-probability -inf now), every clip branch, small and large KL arguments."""
    lp = torch.tensor([-1.0, -1.0, -1.0, -1.0, -math.inf, -2.0, -2.0, -2.0, -0.5, -0.5])
    old = torch.tensor([-1.5, -1.5, -0.5, -0.5, -3.0, -2.0, 98.0, -2.0, -0.5, -0.5])
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, 0.0, -1.0, 2.0, 1.0, -1.0])
    check_policy(lp, old, adv, dev)
    q = torch.tensor([0.0, 1e-6, -1e-3, 0.1, 0.99, 1.01, -5.0, 8.0, -0.999, 1.0])
    lp[4] = -1.0
    check_policy(lp, old, adv, dev, ref=lp + q, kl=0.5)
    assert torch.isfinite(ag.policy_loss(lp.to(dev), (lp - 200).to(dev), torch.zeros(10, device=dev))[0])


def preference_reference(lp, ref, mask, offsets, beta, smoothing, average):
    M, S = lp.numel(), len(offsets) - 1
    seq = sequences(offsets, M)
    live = (seq >= 0) & (mask.bool() if mask is not None else True)
    h, n = torch.zeros(S, dtype=torch.float64), torch.bincount(seq[live], minlength=S).double()
    h.index_add_(0, seq[live], lp.double()[live] - ref.double()[live])
    unit = 1.0 / n.clamp(min=1) if average else torch.ones_like(n)
    h = (h * unit).requires_grad_(True)
    z = beta * (h[0::2] - h[1::2])
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * ls(z) - smoothing * ls(-z)).mean()
    (dh,) = torch.autograd.grad(loss, [h])
    dl = torch.zeros(M, dtype=torch.float64)
    dl[live] = (dh * unit)[seq[live]]
    return loss.detach(), beta * h.detach(), dl


def check_preference(lp, ref, offsets, dev, mask=None, beta=0.1, smoothing=0.0, average=False, index=torch.int32):
    a = lp.to(dev).requires_grad_(True)
    off = torch.tensor(offsets, dtype=index).to(dev)
    beta, smoothing = (float(torch.tensor(v, dtype=torch.float32)) for v in (beta, smoothing))       # float32 arguments
    kw = dict(mask=mask.to(dev) if mask is not None else None, beta=beta, label_smoothing=smoothing, average=average)
    loss, rewards = ag.preference_loss(a, ref.to(dev), off, **kw)
    assert loss.shape == () and not rewards.requires_grad
    (dl,) = torch.autograd.grad(loss * 2.0, [a])
    w_loss, w_rewards, w_dl = preference_reference(lp, ref, mask, offsets, beta, smoothing, average)
    # float64 up to the stores; long sums of float32 terms keep 2^-52 of their terms' size
    size = torch.nan_to_num(lp.double()).abs().sum() + torch.nan_to_num(ref.double()).abs().sum()
    slack = beta * size * 2.0 ** -44
    close(loss, w_loss, 2 * U * w_loss.abs() + slack, "preference loss")
    close(rewards, w_rewards, 2 * U * w_rewards.abs() + slack, "rewards")
    close(dl, 2.0 * w_dl, 8 * U * w_dl.abs() + beta * slack + 1e-44, "preference gradient")
    with torch.no_grad():
        again = ag.preference_loss(a, ref.to(dev), off, **kw)
        assert torch.equal(again[0], loss) and torch.equal(again[1], rewards)


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("P, M", [(1, 2), (1, 5000), (3, 40), (16, 1024), (32, 9000), (33, 9001), (200, 30000), (1500, 2000), (10000, 70000)])
def test_preference_loss(dev, average, P, M):
    lp = -rnd(P, M).abs()
    ref = lp + 0.2 * rnd(P + 1, M)
    mask = torch.rand(M, generator=torch.Generator().manual_seed(M)) < 0.7
    off = ragged(2 * P, 2 * P, M)
    bad = sequences(off, M) < 0
    lp2 = lp.clone()
    lp2[bad] = math.nan
    check_preference(lp2, ref, off, dev, average=average)
    off = ragged(2 * P + 1, 2 * P, M)
    lp2 = lp.clone()
    lp2[~mask] = math.inf
    check_preference(lp2, ref, off, dev, mask=mask, beta=0.5, smoothing=0.1, average=average, index=torch.int64)


def test_preference_loss_extremes(dev):
    M = 64
    lp, ref = -rnd(1, M).abs(), -rnd(2, M).abs()
    check_preference(lp, ref, [0, 0, 0], dev)                                    # two empty sequences: log 2, no gradient
    check_preference(lp, ref, [0, 10, 10], dev)
    check_preference(lp, ref, [0, 30, 64], dev, mask=torch.zeros(M, dtype=torch.uint8))
    big = lp.clone()
    big[:30] += 2000.0
    check_preference(big, ref, [0, 30, 64], dev, smoothing=0.2)                  # saturated, right and wrong way round
    check_preference(big, ref, [0, 0, 64], dev, smoothing=0.5)
    check_preference(-big, ref, [0, 30, 64], dev)
    for at in (5, 40):                                                           # an impossible draw, preferred or rejected: z = -inf or inf
        for smoothing in (0.0, 0.2):
            off = torch.tensor([0, 30, 64], device=dev)
            a = lp.clone()
            a[at] = -math.inf
            a = a.to(dev).requires_grad_(True)
            loss, _ = ag.preference_loss(a, ref.to(dev), off, beta=0.5, label_smoothing=smoothing)
            (dl,) = torch.autograd.grad(loss, [a])
            z = -math.inf if at == 5 else math.inf
            assert float(loss) == (math.inf if at == 5 or smoothing else 0.0)
            dz = 0.5 * (1 / (1 + math.exp(-max(z, -700.0))) - (1 - smoothing))      # exp(700) is finite, its sigmoid below 1e-300
            close(dl, torch.where(torch.arange(M) < 30, dz, -dz), 2 * U * abs(dz) + 1e-44, "gradient of an impossible draw")
    e = torch.empty(0, device=dev, requires_grad=True)
    loss, rewards = ag.preference_loss(e, e.detach(), torch.zeros(5, dtype=torch.int64, device=dev))
    assert abs(float(loss) - math.log(2)) <= 2 * U and torch.equal(rewards, torch.zeros(4, device=dev))


# ------------------------------------------------------------------ together
def fine_tuning_step(p, batch, dtype):
    """embedding -> norm -> head -> log-probability -> both losses; the gradients of every parameter."""
    h = ag.token_embedding(p["emb"], batch["tokens"], scale=4.0, padding_idx=0)
    h = ag.layer_norm(h, p["gamma"], p["beta"])
    logits = ag.linear(h.float(), p["W"], p["b"]).to(dtype)
    lp = ag.class_log_prob(logits, batch["classes"])
    mask = batch["classes"] != -100
    policy, stats = ag.policy_loss(lp, batch["old"], batch["adv"], offsets=batch["offsets"], mask=mask, ref_log_prob=batch["ref"],
                                   kl_coef=0.05, reduction="sequence")
    preference, rewards = ag.preference_loss(lp, batch["ref"], batch["offsets"], mask=mask, beta=0.3)
    loss = policy + preference
    return [loss.detach(), stats, rewards, *torch.autograd.grad(loss, list(p.values()))]


def fine_tuning_setup(dev, dtype, seed=0, n=900, C=211, w=48, V=37, S=6):
    g = torch.Generator().manual_seed(seed)
    put = lambda t: t.to(dtype).to(dev).requires_grad_(True)  # noqa: E731
    p = dict(emb=put(torch.randn(C, w, generator=g) / 4), gamma=put(1 + 0.1 * torch.randn(w, generator=g)), beta=put(0.1 * torch.randn(w, generator=g)),
             W=(0.3 * torch.randn(V, w, generator=g)).to(dev).requires_grad_(True), b=(0.1 * torch.randn(V, generator=g)).to(dev).requires_grad_(True))
    classes = torch.randint(0, V, (n,), generator=g)
    classes[torch.rand(n, generator=g) < 0.2] = -100
    batch = dict(tokens=torch.randint(0, C, (n,), generator=g).to(dev), classes=classes.to(dev), offsets=torch.tensor([0, 100, 100, 450, 460, 700, 890][:S + 1], dtype=torch.int32).to(dev),
                 adv=torch.randn(S, generator=g).to(dev))
    with torch.no_grad():
        h = ag.layer_norm(ag.token_embedding(p["emb"], batch["tokens"], scale=4.0), p["gamma"], p["beta"])
        lp = ag.class_log_prob(ag.linear(h.float(), p["W"], p["b"]).to(dtype), batch["classes"])
        batch["old"] = lp + 0.1 * torch.randn(n, generator=g).to(dev)
        batch["ref"] = lp + 0.1 * torch.randn(n, generator=g).to(dev)
    return p, batch


def test_fine_tuning_step_against_differences(dev):
    """The whole chain's gradient along a direction against central differences of its own forward: a float32 loss of about 1
    with steps of 2e-3 resolves a slope to about 4 u / 2e-3 = 1.2e-4; the slopes here are of order 0.1 to 1, and no ratio may
    cross a border of the clip range, so the clip is opened."""
    p, batch = fine_tuning_setup(dev, torch.float32)

    def f(q):
        h = ag.layer_norm(ag.token_embedding(q["emb"], batch["tokens"], scale=4.0, padding_idx=0), q["gamma"], q["beta"])
        lp = ag.class_log_prob(ag.linear(h, q["W"], q["b"]), batch["classes"])
        mask = batch["classes"] != -100
        a, _ = ag.policy_loss(lp, batch["old"], batch["adv"], offsets=batch["offsets"], mask=mask, ref_log_prob=batch["ref"], clip_low=1.0,
                              clip_high=100.0, kl_coef=0.05, reduction="sequence")
        b, _ = ag.preference_loss(lp, batch["ref"], batch["offsets"], mask=mask, beta=0.3)
        return a + b

    grads = dict(zip(p, torch.autograd.grad(f(p), list(p.values()))))
    for name in p:
        v = torch.randn(p[name].shape, generator=torch.Generator().manual_seed(5)).to(dev)
        if name == "emb":
            v[0] = 0.0                                   # the padding row: used, and without a gradient by definition
        v /= v.norm()
        step = 2e-3 / max(1e-3, float((grads[name] * v).sum().abs())) if name != "emb" else 2e-2
        step = min(step, 2e-2)
        with torch.no_grad():
            up = float(f({**p, name: p[name] + step * v}).double())
            down = float(f({**p, name: p[name] - step * v}).double())
        slope = float((grads[name].double() * v.double()).sum())
        scale = float(grads[name].double().norm())
        # 4 u of a loss of size |f| over the step, and the third derivative's share: step^2 of the gradient's size, tenfold
        tol = 8 * U * max(1.0, abs(up)) / step + 10 * step * step * scale + 1e-3 * abs(slope)
        assert abs((up - down) / (2 * step) - slope) <= tol, (name, (up - down) / (2 * step), slope, tol)


def test_policy_step_of_the_denoiser(dev):
    """A node tower's attribute draws: at ratio 1 and advantage 1 the policy loss is -1 and has the gradient of the mean cross
    entropy, which softmax_ce2 gives for the same logits.  The two logit gradients differ by a few roundings of each element
    and go through the same backward kernels: 64 u of each sum's terms, taken as 64 times the largest gradient."""
    import graphmaker_amd as gm
    from graphmaker_amd import ops
    torch.manual_seed(0)
    n, F, Y = 90, 12, 4
    tower = gm.GNNTower(num_attrs_X=F, num_classes_X=2, num_classes_Y=Y, hidden_t=8, hidden_X=32, hidden_Y=16, out_size=2 * F,
                        num_gnn_layers=2, dropout=0.0, node_mode=True).to(dev).train()
    E = (torch.rand(n, n, generator=torch.Generator().manual_seed(1)) < 0.1).long().triu(1)
    adj = ops.adjacency_from_bitmap(ops.bitmap_from_dense((E + E.t()).to(dev)), n)
    g = torch.Generator().manual_seed(2)
    x_t, drawn = (torch.randint(0, 2, (n, F), generator=g) for _ in range(2))
    X = torch.nn.functional.one_hot(x_t, 2).float().reshape(n, -1).to(dev)
    labels = torch.randint(0, Y, (n,), generator=g).to(dev)
    t = torch.tensor([0.5], device=dev)
    logits = tower(t, X, labels, adj)
    ce = ag.softmax_ce2(logits.reshape(-1, 2), drawn.to(torch.uint8).reshape(-1).to(dev))
    want = torch.autograd.grad(ce, list(tower.parameters()))
    lp = ag.class_log_prob(tower(t, X, labels, adj), drawn.to(dev))
    assert lp.shape == (n, F)
    loss, stats = ag.policy_loss(lp, lp.detach(), torch.ones(1, device=dev), offsets=torch.tensor([0, n * F], device=dev))
    got = torch.autograd.grad(loss, list(tower.parameters()))
    assert abs(float(loss.detach()) + 1.0) <= 2 * U and stats.tolist()[2:] == [0.0, float(n * F)]
    for (name, _), a, b in zip(tower.named_parameters(), got, want):
        close(a, b.cpu(), 64 * 64 * U * b.abs().max().item() + 1e-9, name)


@pytest.mark.parametrize("dt", TYPES)
def test_fine_tuning_step_is_reproducible_on_any_stream(dev, dt):
    p, batch = fine_tuning_setup(dev, DT[dt])
    want = fine_tuning_step(p, batch, DT[dt])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:                                    # both steps in flight at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(fine_tuning_step(p, batch, DT[dt]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(out, want):
            assert torch.isfinite(b).all() and torch.equal(a, b)


def test_fine_tuning_step_in_a_graph(dev):
    """Two captured steps of different inputs that share a memory pool, replayed in turn with eager work between."""
    steps = [fine_tuning_setup(dev, torch.bfloat16, seed=s, S=s + 4 if s % 2 == 0 else 6) for s in (0, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for p, b in steps:
            fine_tuning_step(p, b, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for p, b in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(fine_tuning_step(p, b, torch.bfloat16))
        graphs.append(g)
    for turn in range(4):
        for k in (0, 1):
            p, b = steps[k]
            b["tokens"].copy_((b["tokens"] * 7 + turn) % 211)
            b["classes"].copy_(torch.where(b["classes"] < 0, b["classes"], (b["classes"] + turn) % 37))
            torch.cuda.synchronize()
            want = fine_tuning_step(p, b, torch.bfloat16)
            graphs[k].replay()
            torch.cuda.synchronize()
            for got, w in zip(outs[k], want):
                assert torch.equal(got, w), (turn, k)


def test_capture_beside_a_living_eager_graph_is_refused(dev):
    """Refused before anything is captured; fine once the eager graph is gone, and with leaves that it does not hold."""
    x, w = rnd(1, 30, 64).to(dev), (1 + 0.1 * rnd(2, 64)).to(dev).requires_grad_(True)
    emb = rnd(3, 40, 64).to(dev).requires_grad_(True)
    tok = torch.arange(30, device=dev)
    alive = ag.layer_norm(x, w)                          # recorded eagerly on the default stream
    held = ag.token_embedding(emb, tok)
    torch.cuda.synchronize()
    fresh = rnd(4, 30, 64).to(dev).requires_grad_(True)
    for call in (lambda: ag.layer_norm(x, w), lambda: ag.token_embedding(emb, tok),
                 lambda: ag.layer_norm(fresh * 2, w), lambda: ag.layer_norm(fresh, None, w)):
        with pytest.raises(RuntimeError, match="same leaf tensor is alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive, held
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ag.layer_norm(x, w)
        y = y + ag.layer_norm(y, w)                      # the same leaf twice inside the capture
        (dw,) = torch.autograd.grad(y.sum(), [w])
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        z = ag.layer_norm(x, w)
        z = z + ag.layer_norm(z, w)
        assert torch.equal(z, y) and torch.equal(torch.autograd.grad(z.sum(), [w])[0], dw)


def test_upstream_gradients_and_inplace_loss(dev):
    """The losses are ordinary scalars: scaled in place, summed, used twice, or not used at all."""
    lp, old, _ = (t.to(dev) for t in ratios(4, 500))
    a = lp.clone().requires_grad_(True)
    loss, _ = ag.policy_loss(a, old, rnd(1, 500).to(dev))
    (g1,) = torch.autograd.grad(loss, [a], retain_graph=True)
    (g2,) = torch.autograd.grad(loss, [a], torch.tensor(0.5, device=dev), retain_graph=True)
    assert torch.allclose(g1 * 0.5, g2, rtol=4 * U, atol=0)
    (g3,) = torch.autograd.grad(loss, [a])
    assert torch.equal(g1, g3)
    loss, _ = ag.policy_loss(a, old, rnd(1, 500).to(dev))
    loss /= 4
    (g4,) = torch.autograd.grad(loss, [a])
    assert torch.equal(g1 / 4, g4)                       # a power of two


@pytest.mark.parametrize("S, M", [(8192, 9000), (8194, 9000), (300000, 400001), (1200000, 700000)])
def test_losses_of_many_short_sequences(dev, S, M):
    """More sequences than one workgroup takes: the totals and the weights come from several."""
    lp, old, ref = ratios(S, M)
    mask = torch.rand(M, generator=torch.Generator().manual_seed(S)) < 0.8
    off = ragged(S + 1, S, M)
    for reduction in ("token", "sequence"):
        check_policy(lp, old, rnd(S, S), dev, ref=ref, mask=mask, offsets=off, kl=0.05, reduction=reduction)
    check_preference(lp, ref, off, dev, mask=mask, beta=0.3, smoothing=0.1, average=True)


@pytest.mark.parametrize("C", [5, 200])
def test_token_embedding_without_tokens_and_of_one(dev, C):
    W = rnd(1, C, 24).to(dev).requires_grad_(True)
    for shape in ((0,), (3, 0)):
        y = ag.token_embedding(W, torch.empty(shape, dtype=torch.int64, device=dev))
        assert y.shape == shape + (24,)
        (dW,) = torch.autograd.grad(y.sum(), [W])
        assert not dW.any()
    y = ag.token_embedding(W, torch.tensor(C - 1, device=dev), scale=2.0)        # no dimension
    assert y.shape == (24,) and torch.equal(y, 2 * W.detach()[C - 1])
    (dW,) = torch.autograd.grad(y.sum(), [W])                                    # the gradient of a sum: one element, expanded
    assert (dW[C - 1] == 2).all() and not dW[:C - 1].any()
    y = ag.token_embedding(W, torch.arange(C, device=dev)) + ag.token_embedding(W, torch.arange(C, device=dev).flip(0))
    assert (torch.autograd.grad(y.sum(), [W])[0] == 2).all()                     # the same table twice


def test_single_rows_and_inference_mode(dev):
    x = rnd(1, 70).to(dev).requires_grad_(True)
    gamma, beta = rnd(2, 70).to(dev).requires_grad_(True), rnd(3, 70).to(dev)
    got = torch.autograd.grad(ag.layer_norm(x, gamma, beta).sum(), [x, gamma])
    rows = ag.layer_norm(x[None], gamma, beta)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(rows.sum(), [x, gamma])))
    lp = ag.class_log_prob(x, torch.tensor(9, device=dev))                       # one row, a class without a dimension
    assert lp.shape == () and torch.equal(lp, ag.class_log_prob(x[None], torch.tensor([9], device=dev))[0])
    (dx,) = torch.autograd.grad(lp, [x])
    close(dx, torch.nn.functional.one_hot(torch.tensor(9), 70).double() - x.detach().cpu().double().softmax(0), (D(70) + 8) * U, "one row")
    with torch.inference_mode():
        y = ag.layer_norm(x, gamma, beta)
        assert not y.requires_grad and torch.equal(y, rows[0])
        assert torch.equal(ag.class_log_prob(x, torch.tensor(9, device=dev)), lp)
        loss, _ = ag.policy_loss(y, y, y)
        assert not loss.requires_grad
    e = torch.empty(0, 70, device=dev, requires_grad=True)
    got = torch.autograd.grad(ag.layer_norm(e, gamma, beta).sum(), [e, gamma])
    assert got[0].shape == (0, 70) and not got[1].any()
    assert ag.class_log_prob(e, torch.empty(0, dtype=torch.int32, device=dev)).shape == (0,)


def test_losses_of_strided_and_many_dimensional_items(dev):
    """Items in a transposed batch: the losses take them in the order of the tensor's indexes."""
    lp = (-rnd(1, 12, 7).abs()).to(dev)
    old, ref, adv = (lp + 0.1 * rnd(k, 12, 7).to(dev) for k in (2, 3, 4))
    mask = rnd(5, 12, 7).to(dev) > 0
    a, b = lp.t().detach().requires_grad_(True), lp.t().contiguous().requires_grad_(True)
    for f in (lambda q: ag.policy_loss(q, old.t(), adv.t(), mask=mask.t(), ref_log_prob=ref.t(), kl_coef=0.1),
              lambda q: ag.preference_loss(q, ref.t(), torch.tensor([0, 9, 9, 50, 84], device=dev), mask=mask.t())):
        x, y = f(a), f(b)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
        assert torch.equal(torch.autograd.grad(x[0], [a])[0], torch.autograd.grad(y[0], [b])[0])


# ------------------------------------------------------------------ sizes past 32 bits
def test_rows_past_2_31_elements(dev):
    M, N = 262_147, 8200                                 # 2.15e9 elements, 4.3 GB in 16 bits
    x = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    tail = rnd(1, 4, N, dtype=torch.bfloat16).to(dev)
    x[-4:] = tail
    assert torch.equal(ag.layer_norm(x)[-4:], ag.layer_norm(tail))
    c = torch.zeros(M, dtype=torch.int64, device=dev)
    c[-4:] = N - 1
    a = x.requires_grad_(True)
    lp = ag.class_log_prob(a, c)
    t = tail.clone().requires_grad_(True)
    tp = ag.class_log_prob(t, c[-4:])
    assert torch.allclose(lp[-4:], tp, rtol=1e-5)
    g = torch.ones(M, device=dev)
    got = torch.autograd.grad(lp, [a], g)[0][-4:]
    assert torch.allclose(got.float(), torch.autograd.grad(tp, [t], g[-4:])[0].float(), rtol=2 * ut(torch.bfloat16), atol=1e-7)
    del lp, got, a, x
    W = rnd(2, 50, N, dtype=torch.bfloat16).to(dev).requires_grad_(True)
    tok = torch.arange(M, device=dev) % 49
    tok[-1] = 49
    y = ag.token_embedding(W, tok)
    assert torch.equal(y[-50:], W.detach()[tok[-50:]])
    up = torch.zeros_like(y)
    up[-1] = 1.5
    (dW,) = torch.autograd.grad(y, [W], up)
    assert torch.equal(dW[49], up[-1]) and not dW[:49].any()
