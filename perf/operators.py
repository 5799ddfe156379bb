"""Measured cases of the token, normalisation and fine-tuning operators of graphmaker_amd.autograd: token_embedding,
layer_norm, class_log_prob, policy_loss and preference_loss, each beside its plain form in elementary torch operations and
its definition in 64 bits.

`own` chooses the side that run() takes: False = the plain form (32 bits whatever the inputs' type, rounded once at the
end; log ratios, long sums and the KL term in 64), True = the library's operators as a training loop or a server calls
them.  A case with grad = True is a training pass (forward and every gradient), one with grad = False a serving pass.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04
BETA, SMOOTHING = 0.1, 0.05


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # eight tokens of a decoding step looked up in a 16-bit table: latency
        dict(name="embed_step", op="embed", n=8, C=32003, w=1024, dtype="bf16", index="i32", skew="zipf", pad=False, grad=False),
        # the label embedding of a 13,752-node graph with 10 classes and 64 columns (this package's largest shipped
        # configuration), forward and gradient: ten rows that take more than a thousand tokens each
        dict(name="embed_labels", op="embed", n=13752, C=10, w=64, dtype="f32", index="i32", skew="uniform", pad=False, grad=True),
        # a padded training batch against a large vocabulary: few rows with thousands of tokens, most with none
        dict(name="embed_vocab", op="embed", n=130941, C=50021, w=1024, dtype="bf16", index="i64", skew="zipf", pad=True, grad=True),
        # the update block's norm over the nodes of the same graph (512 hidden columns), forward and gradient
        dict(name="norm_tower", op="norm", M=13752, N=512, dtype="f32", grad=True),
        # the norm of a few tokens in a decoding step: latency
        dict(name="norm_step", op="norm", M=4, N=4096, dtype="f16", grad=False),
        # the norm of a wide 16-bit model in training
        dict(name="norm_wide", op="norm", M=8191, N=8192, dtype="bf16", grad=True),
        # log-probabilities of the 2,097,152 edge draws of a training batch, two classes
        dict(name="logp_pairs", op="logp", M=2097152, V=2, dtype="f32", grad=True),
        # log-probabilities of a training batch's tokens against a large vocabulary; the last columns are banned
        dict(name="logp_vocab", op="logp", M=4095, V=50021, dtype="bf16", grad=True),
        # the sampled tokens of a decoding step: few long rows
        dict(name="logp_step", op="logp", M=3, V=128256, dtype="f16", grad=False),
        # one clipped policy update on the attribute draws (13,752 x 767 in all) of eight sampled graphs, with the KL term
        dict(name="policy_graph", op="policy", M=10547784, S=8, reduction="token", kl=True, mask=False),
        # a small batch of ragged answers, each answer counted once, prompts masked
        dict(name="policy_answers", op="policy", M=20011, S=64, reduction="sequence", kl=True, mask=True),
        # ragged pairs of answers, prompts masked
        dict(name="prefer_pairs", op="prefer", M=1048576, P=512, mask=True, average=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embed", "norm", "logp", "policy", "prefer"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    grad = rng.random() < 0.7
    if op == "embed":
        w = _log_uniform(rng, 1, 2048)
        C = min(_log_uniform(rng, 1, 65536), max(1, 2 ** 25 // w))
        n = min(_log_uniform(rng, 1, 131072), max(1, 2 ** 25 // w))
        return dict(op=op, n=n, C=C, w=w, dtype=dtype, index=rng.choice(["i32", "i64"]),
                    skew=rng.choice(["zipf", "uniform"]), pad=rng.random() < 0.5, grad=grad)
    if op == "norm":
        N = _log_uniform(rng, 2, 16384)
        return dict(op=op, M=min(_log_uniform(rng, 1, 65536), max(1, 2 ** 25 // N)), N=N, dtype=dtype, grad=grad)
    if op == "logp":
        V = _log_uniform(rng, 2, 131072)
        return dict(op=op, M=min(_log_uniform(rng, 1, 2 ** 21), max(1, 2 ** 25 // V)), V=V, dtype=dtype, grad=grad)
    if op == "policy":
        S = rng.choice([0, 1, _log_uniform(rng, 2, 1024)])
        return dict(op=op, M=_log_uniform(rng, 1, 2 ** 23), S=S,
                    reduction=rng.choice(["token", "sequence"]) if S else "token", kl=rng.random() < 0.5, mask=rng.random() < 0.5)
    P = _log_uniform(rng, 1, 1024)
    return dict(op=op, M=_log_uniform(rng, 2, 2 ** 22), P=P, mask=rng.random() < 0.5, average=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype="f32", scale=1.0, shift=0.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return x.mul_(scale).add_(shift).to(DTYPES[dtype])


def _offsets(rng, M, S):
    """S ragged, consecutive sequences in M items: log-normal lengths, one of 16 empty, and up to 3 % of the items behind
    the last one (the padding of a batch of fixed size)."""
    share = np.exp(rng.normal(0.0, 0.8, S)) * (rng.random(S) >= 1.0 / 16)
    if share.sum() == 0.0:
        share[0] = 1.0
    used = M - int(rng.integers(0, max(1, M // 32) + 1)) if M > 1 else M
    ends = np.round(np.cumsum(share) / share.sum() * used).astype(np.int64)
    return torch.from_numpy(np.concatenate([[0], ends])).to(torch.int32).cuda()


def _prompt_mask(g, M):
    """About a third of the items off, in runs of 16 as prompts and tool answers leave them."""
    runs = torch.rand((M + 15) // 16, generator=g, device="cuda") < 0.67
    return runs.repeat_interleave(16)[:M].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = np.random.default_rng([int(seed), 77])
    s = dict(case)
    op = case["op"]
    if op == "embed":
        n, C, w = case["n"], case["C"], case["w"]
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        if case["skew"] == "zipf":                       # the k-th most frequent token has a share of about 1 / (k log C)
            tok = torch.exp(u * math.log(C + 1)).long() - 1
            tok = torch.randperm(C, generator=g, device="cuda")[tok.clamp_(0, C - 1)]
        else:
            tok = (u * C).long().clamp_(0, C - 1)
        s["padding"] = None
        if case["pad"]:
            s["padding"] = C // 2
            tok[n - n // 8:] = C // 2
        s["tokens"] = tok.to(torch.int32 if case["index"] == "i32" else torch.int64)
        s["weight"] = _randn(g, C, w, dtype=case["dtype"], scale=w ** -0.5).requires_grad_(case["grad"])
        s["scale"] = float(w) ** 0.5
        if case["grad"]:
            s["up"] = _randn(g, n, w, dtype=case["dtype"])
    elif op == "norm":
        M, N = case["M"], case["N"]
        x = torch.randn(M, N, generator=g, device="cuda")
        x.mul_(_randn(g, N, scale=0.3).exp_()).add_(_randn(g, M, 1, scale=0.5))     # channels and rows differ in size
        s["x"] = x.to(DTYPES[case["dtype"]]).requires_grad_(case["grad"])
        s["gamma"] = _randn(g, N, dtype=case["dtype"], scale=0.2, shift=1.0).requires_grad_(case["grad"])
        s["beta"] = _randn(g, N, dtype=case["dtype"], scale=0.2).requires_grad_(case["grad"])
        if case["grad"]:
            s["up"] = _randn(g, M, N, dtype=case["dtype"])
    elif op == "logp":
        M, V = case["M"], case["V"]
        logits = torch.randn(M, V, generator=g, device="cuda").mul_(2.0)
        if V > 4096:
            logits[:, V - 61:] = -math.inf               # columns behind the vocabulary's end, never drawn
        noise = torch.rand(M, V, generator=g, device="cuda").clamp_(1e-20, 1 - 1e-7)
        cls = noise.log_().neg_().log_().neg_().add_(logits).argmax(1)
        del noise
        cls[torch.rand(M, generator=g, device="cuda") < 0.05] = IGNORE
        s["classes"] = cls
        s["logits"] = logits.to(DTYPES[case["dtype"]]).requires_grad_(case["grad"])
        if case["grad"]:
            s["up"] = _randn(g, M)
    else:
        M = case["M"]
        lp = _randn(g, M).abs_().mul_(-1.5)
        s["log_prob"] = lp.clone().requires_grad_(True)
        s["ref"] = lp + _randn(g, M, scale=0.1)
        s["mask"] = _prompt_mask(g, M) if case["mask"] else None
        if op == "policy":
            d = _randn(g, M, scale=0.15)
            # the gradient jumps where the ratio meets a border of the clip range: no ratio within 1e-4 of one, where
            # the rounding of the inputs' own difference decides
            for b in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
                d = torch.where((d - b).abs() < 1e-4, d + 3e-4, d)
            s["old"] = lp - d
            s["offsets"] = _offsets(rng, M, case["S"]) if case["S"] else None
            s["advantage"] = _randn(g, case["S"] or M)
            if not case["kl"]:
                s["ref"] = None
        else:
            s["offsets"] = _offsets(rng, M, 2 * case["P"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"embed": _embed, "norm": _norm, "logp": _logp, "policy": _policy, "prefer": _prefer}[op](s)


def _run_own(s):
    from graphmaker_amd import autograd as ag

    op = s["op"]
    if op == "embed":
        y = ag.token_embedding(s["weight"], s["tokens"], scale=s["scale"], padding_idx=s["padding"])
        return [y.detach(), *torch.autograd.grad(y, [s["weight"]], s["up"])] if s["grad"] else [y]
    if op == "norm":
        y = ag.layer_norm(s["x"], s["gamma"], s["beta"])
        return [y.detach(), *torch.autograd.grad(y, [s["x"], s["gamma"], s["beta"]], s["up"])] if s["grad"] else [y]
    if op == "logp":
        y = ag.class_log_prob(s["logits"], s["classes"], ignore_index=IGNORE)
        return [y.detach(), *torch.autograd.grad(y, [s["logits"]], s["up"])] if s["grad"] else [y]
    if op == "policy":
        loss, stats = ag.policy_loss(s["log_prob"], s["old"], s["advantage"], offsets=s["offsets"], mask=s["mask"],
                                     ref_log_prob=s["ref"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                                     kl_coef=KL if s["kl"] else 0.0, reduction=s["reduction"])
        return [loss.detach(), stats, *torch.autograd.grad(loss, [s["log_prob"]])]
    loss, rewards = ag.preference_loss(s["log_prob"], s["ref"], s["offsets"], mask=s["mask"], beta=BETA,
                                       label_smoothing=SMOOTHING, average=s["average"])
    return [loss.detach(), rewards, *torch.autograd.grad(loss, [s["log_prob"]])]


def _embed(s):
    weight, tok = s["weight"], s["tokens"].long()
    y = (weight[tok].float() * s["scale"]).to(weight.dtype)
    if not s["grad"]:
        return [y]
    g = s["up"].float()
    if s["padding"] is not None:
        g = g * (tok != s["padding"])[:, None]
    dw = torch.zeros(weight.shape, dtype=torch.float32, device=g.device).index_add_(0, tok, g)
    return [y, (dw * s["scale"]).to(weight.dtype)]


def _norm(s):
    x, gamma, beta = s["x"].float(), s["gamma"].float(), s["beta"].float()
    dt = s["x"].dtype
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * gamma + beta).to(dt)
    if not s["grad"]:
        return [y]
    g = s["up"].float()
    gg = g * gamma
    dx = rstd * (gg - gg.mean(1, keepdim=True) - xh * (gg * xh).mean(1, keepdim=True))
    return [y, dx.to(dt), (g * xh).sum(0).to(dt), g.sum(0).to(dt)]


def _logp(s):
    x, cls = s["logits"].float(), s["classes"].long()
    live = cls != IGNORE
    at = torch.where(live, cls, 0)[:, None]
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(1, keepdim=True)
    lp = torch.where(live, (x.gather(1, at) - torch.log(z))[:, 0], 0.0)
    if not s["grad"]:
        return [lp]
    g = torch.where(live, s["up"], 0.0)[:, None]
    return [lp, (e / z * -g).scatter_add_(1, at, g).to(s["logits"].dtype)]


def _sequence_of(offsets, M):
    """(sequence of each item, whether it is inside one)."""
    seq = torch.bucketize(torch.arange(M, device=offsets.device), offsets.long()[1:], right=True)
    return seq.clamp(max=offsets.numel() - 2), seq < offsets.numel() - 1


def _policy(s):
    lp, old = s["log_prob"], s["old"]
    M = lp.numel()
    live = torch.ones(M, dtype=torch.bool, device=lp.device) if s["mask"] is None else s["mask"]
    adv = s["advantage"]
    if s["offsets"] is not None:
        seq, inside = _sequence_of(s["offsets"], M)
        live = live & inside
        adv = adv[seq]
    if s["reduction"] == "token":
        weight = live / live.sum().clamp(min=1)
    else:
        count = torch.zeros(s["offsets"].numel() - 1, dtype=torch.float64, device=lp.device).index_add_(0, seq, live.double())
        weight = torch.where(live, (1.0 / (count.clamp(min=1.0) * (count > 0).sum().clamp(min=1)))[seq], 0.0)
    r = torch.exp(lp.double() - old.double())
    low, high = r < 1.0 - CLIP_LOW, r > 1.0 + CLIP_HIGH
    cut = ((adv > 0) & high) | ((adv < 0) & low)
    surrogate = -torch.where(cut, r.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH), r) * adv
    dlp = torch.where(cut, 0.0, -adv * r)
    kl = torch.zeros_like(r)
    if s["kl"]:
        d = s["ref"].double() - lp.double()
        kl = torch.exp(d) - d - 1.0
        dlp = dlp + KL * (1.0 - torch.exp(d))
    weight = weight.double()
    means = [(weight * v).sum() for v in (surrogate, kl, cut.double())]
    stats = torch.stack(means + [live.sum().double()]).float()
    return [(means[0] + KL * means[1]).float(), stats, (weight * dlp).float()]


def _prefer(s):
    lp = s["log_prob"]
    M, S = lp.numel(), s["offsets"].numel() - 1
    seq, live = _sequence_of(s["offsets"], M)
    if s["mask"] is not None:
        live = live & s["mask"]
    d = torch.where(live, lp.double() - s["ref"].double(), 0.0)
    h = torch.zeros(S, dtype=torch.float64, device=lp.device).index_add_(0, seq, d)
    unit = torch.ones_like(h)
    if s["average"]:
        unit = 1.0 / torch.zeros_like(h).index_add_(0, seq, live.double()).clamp(min=1.0)
    h = h * unit
    z = BETA * (h[0::2] - h[1::2])
    up = torch.clamp(-z, min=0) + torch.log1p(torch.exp(-z.abs()))          # -log sigmoid(z)
    loss = ((1.0 - SMOOTHING) * up + SMOOTHING * (up + z)).mean()
    dz = (1.0 / (1.0 + torch.exp(-z)) - (1.0 - SMOOTHING)) / z.numel()
    dh = torch.stack([BETA * dz, -BETA * dz], 1).reshape(-1) * unit
    return [loss.float(), (BETA * h).float(), torch.where(live, dh[seq], 0.0).float()]


# ------------------------------------------------------------------ what a pass cannot do without
def _touched(C, n, skew):
    """Expected number of different rows among n tokens."""
    k = np.arange(1, C + 1, dtype=np.float64)
    p = np.log((k + 1) / k) / math.log(C + 1) if skew == "zipf" else np.full(C, 1.0 / C)
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    op = case["op"]
    if op == "embed":
        n, C, w, e = case["n"], case["C"], case["w"], BYTES[case["dtype"]]
        size = n * (4 if case["index"] == "i32" else 8) + (_touched(C, n, case["skew"]) + n) * w * e
        return dict(bytes=size + ((n + C) * w * e if case["grad"] else 0), flops=n * w * (2 if case["grad"] else 1))
    if op == "norm":
        M, N, e = case["M"], case["N"], BYTES[case["dtype"]]
        if not case["grad"]:
            return dict(bytes=2 * (M + 1) * N * e, flops=8 * M * N)
        return dict(bytes=(4 * M + 4) * N * e, flops=22 * M * N)
    if op == "logp":
        M, V, e = case["M"], case["V"], BYTES[case["dtype"]]
        if not case["grad"]:
            return dict(bytes=M * V * e + 12 * M, flops=4 * M * V)
        return dict(bytes=2 * M * V * e + 16 * M, flops=8 * M * V)
    M = case["M"]
    if op == "policy":
        return dict(bytes=M * (12 + (4 if case["kl"] else 0) + (1 if case["mask"] else 0)) + (8 * case["S"] or 4 * M),
                    flops=M * (20 if case["kl"] else 10))
    return dict(bytes=M * (12 + (1 if case["mask"] else 0)) + 16 * case["P"], flops=4 * M)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if case["op"] == "embed":
            table, ids = s["weight"].to(f64), s["tokens"].to(torch.int64)
            looked = table.index_select(0, ids) * s["scale"]
            if not case["grad"]:
                return [looked]
            grad = torch.zeros_like(table)
            keep = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids.ne(s["padding"])
            grad.index_put_((ids[keep],), s["up"][keep].to(f64) * s["scale"], accumulate=True)
            return [looked, grad]
        if case["op"] == "norm":
            outs = [[], []]
            dgamma, dbeta = (torch.zeros(case["N"], dtype=f64, device="cuda") for _ in range(2))
            gamma, beta = s["gamma"].to(f64), s["beta"].to(f64)
            step = max(1, 2 ** 24 // case["N"])
            for a in range(0, case["M"], step):
                x = s["x"][a:a + step].to(f64)
                var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
                sigma = (var + 1e-5).sqrt()
                u = (x - mean) / sigma
                outs[0].append(torch.addcmul(beta, u, gamma))
                if case["grad"]:
                    dy = s["up"][a:a + step].to(f64)
                    dgamma += torch.linalg.vecdot(dy, u, dim=0)
                    dbeta += dy.sum(0)
                    du = dy * gamma
                    along = torch.linalg.vecdot(du, u).unsqueeze(1) / case["N"]
                    outs[1].append((du - du.mean(1, keepdim=True) - along * u) / sigma)
            return [torch.cat(outs[0])] + ([torch.cat(outs[1]), dgamma, dbeta] if case["grad"] else [])
        if case["op"] == "logp":
            lps, grads = [], []
            step = max(1, 2 ** 24 // case["V"])
            for a in range(0, case["M"], step):
                x, c = s["logits"][a:a + step].to(f64), s["classes"][a:a + step]
                rows = torch.nonzero(c != IGNORE)[:, 0]
                full = x - torch.logsumexp(x, 1, keepdim=True)
                lp = torch.zeros(len(c), dtype=f64, device="cuda")
                lp[rows] = full[rows, c[rows]]
                lps.append(lp)
                if case["grad"]:
                    up = s["up"][a:a + step].to(f64)
                    grad = torch.zeros_like(x)
                    grad[rows] = -up[rows, None] * full[rows].exp()
                    grad[rows, c[rows]] += up[rows]
                    grads.append(grad)
            return [torch.cat(lps)] + ([torch.cat(grads)] if case["grad"] else [])
        M = case["M"]
        alive = torch.ones(M, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"].clone()
        if s["offsets"] is not None:
            ends = s["offsets"].to(torch.int64)
            length = ends[1:] - ends[:-1]
            owner = torch.repeat_interleave(torch.arange(length.numel(), device="cuda"), length)
            alive[owner.numel():] = False
            owner = torch.nn.functional.pad(owner, (0, M - owner.numel()))
            living = torch.bincount(owner[alive], minlength=length.numel()).to(f64)
        picked = torch.nonzero(alive)[:, 0]
        lp = s["log_prob"][picked].to(f64)
        dlp = torch.zeros(M, dtype=f64, device="cuda")
        if case["op"] == "policy":
            A = s["advantage"].to(f64)
            A = A[picked] if s["offsets"] is None else A[owner[picked]]
            if case["reduction"] == "token":
                share = torch.full_like(lp, 1.0 / max(1, picked.numel()))
            else:
                share = 1.0 / living[owner[picked]] / max(1, int((living > 0).sum()))
            ratio = (lp - s["old"][picked].to(f64)).exp()
            kept, clipped = ratio * A, ratio.clip(1 - CLIP_LOW, 1 + CLIP_HIGH) * A
            bound = clipped < kept
            gain = torch.minimum(kept, clipped)
            slope = torch.where(bound, torch.zeros_like(kept), kept)
            apart = torch.zeros_like(kept)
            if case["kl"]:
                gap = s["ref"][picked].to(f64) - lp
                apart = torch.special.expm1(gap) - gap
                slope = slope + KL * torch.special.expm1(gap)
            dlp[picked] = -share * slope
            part = [-(share @ gain), share @ apart, share @ bound.to(f64)]
            stats = torch.stack(part + [torch.tensor(float(picked.numel()), dtype=f64, device="cuda")])
            return [part[0] + KL * part[1], stats, dlp]
        gap = lp - s["ref"][picked].to(f64)
        total = torch.cumsum(torch.zeros(M, dtype=f64, device="cuda").index_copy_(0, picked, gap), 0)
        total = torch.nn.functional.pad(total, (1, 0))
        h = total[ends[1:]] - total[ends[:-1]]
        if case["average"]:
            h = h / living.clamp(min=1)
        better, worse = h.view(-1, 2).unbind(1)
        margin = BETA * (better - worse)
        ls = torch.nn.functional.logsigmoid
        loss = -((1 - SMOOTHING) * ls(margin) + SMOOTHING * ls(-margin)).mean()
        slope = (SMOOTHING * torch.sigmoid(margin) - (1 - SMOOTHING) * torch.sigmoid(-margin)) * BETA / margin.numel()
        each = torch.stack([slope, -slope], 1).view(-1)
        if case["average"]:
            each = each / living.clamp(min=1)
        dlp[picked] = each[owner[picked]]
        return [loss, BETA * h, dlp]
