"""The tape of the training step (reference: log_p_t, model/diffusion.py:606-654, :1035-1094, driven by
train_sync.py:94-120 / train_async.py).  torch.autograd only records the operator graph; every forward and every
gradient below is one or a few calls into libgraphmaker_hip.so (gm_train.hip, gm_gemm.hip, gm_nodeops.hip).  All
reductions run in a fixed order, so a step is reproducible run to run.

Operators (each a torch.autograd.Function over contiguous float32 device tensors):
    linear(x, W, b, relu)            nn.Linear (+ReLU)                         model/gnn.py:116-126,138-142,226-230
    update_block(x, W, b, g, beta)   Linear -> ReLU -> LayerNorm               model/gnn.py:27-38
    spmm_mean(adj, H)                A @ H with A = D^-1 A                     model/gnn.py:60-61
    embedding(weight, idx)           nn.Embedding                              model/gnn.py:155
    hadamard_gather(h, src, dst)     h[src] * h[dst]                           model/gnn.py:246
    softmax_ce2(logits, target)      F.cross_entropy, 2 classes, mean          model/diffusion.py:139,513
    dropout(x, p, seed, call)        nn.Dropout in training mode               model/gnn.py:31,37

Operators for wider models, large vocabularies and fine-tuning on rewards or preferences (no counterpart in the reference;
float32, bfloat16 or float16 rows, sums in float32 or float64):
    token_embedding(weight, tokens, scale, padding_idx)            scaled lookup; gradient by sorted tokens
    layer_norm(x, gamma, beta, eps)                                layer norm over rows of any width
    class_log_prob(logits, classes, ignore_index)                  log-probability of one class a row
    policy_loss(log_prob, old_log_prob, advantage, ...)            clipped policy loss with a KL term
    preference_loss(log_prob, ref_log_prob, offsets, ...)          loss of preferred over rejected sequences
They enqueue on the current stream of their tensors' device, keep their workspaces to one call, read nothing back to the
host and can be captured in a HIP graph, forward and backward.  Capture a backward pass only when no graph recorded eagerly
over the same leaf tensors is still alive: torch ties a leaf's gradient accumulation to the stream of the first such graph.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops
from ._lib import F32, I32, I64, U32, U64, ptr, require, stream_ptr

_scratch_bufs = {}


def _scratch(nbytes, device, slot=0):
    """Device scratch for split-K / block partials.  One buffer per (device, slot), grown on demand; kernels that use
    it run back to back on the current stream, so sharing is safe."""
    key = (device, slot)
    buf = _scratch_bufs.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)
        _scratch_bufs[key] = buf
    return buf


def _c(t):
    return t if t.is_contiguous() else t.contiguous()


def C_void(t, offset_elems):
    """Pointer to element `offset_elems` of a float32 tensor."""
    return ctypes.c_void_p(t.data_ptr() + 4 * offset_elems)


def gemm(a_red, b_red, M, N, K, A, lda, B, ldb, *, bias=None, mask=None, relu=False, out=None):
    """gm_gemm: C[m][n] = act(sum_k a(m,k) b(n,k) + bias[n]) (zero where mask <= 0)."""
    dev = A.device
    C_ = out if out is not None else torch.empty((M, N), dtype=torch.float32, device=dev)
    need = L.load().gm_gemm_workspace_bytes(I64(M), I64(N), I64(K))
    ws = _scratch(need, dev) if need else None
    L.call("gm_gemm", I32(int(a_red)), I32(int(b_red)), I64(M), I64(N), I64(K), ptr(A), I64(lda), ptr(B), I64(ldb), ptr(bias),
           ptr(mask), I64(N if mask is not None else 0), I32(int(relu)), ptr(C_), I64(N), ptr(ws), I64(ws.numel() if ws is not None else 0),
           stream_ptr())
    return C_


def colsum(X):
    M, N = X.shape
    out = torch.empty(N, dtype=torch.float32, device=X.device)
    need = L.load().gm_colsum_workspace_bytes(I64(M), I64(N))
    ws = _scratch(need, X.device)
    L.call("gm_colsum", I64(M), I64(N), ptr(X), I64(N), ptr(out), ptr(ws), I64(ws.numel()), stream_ptr())
    return out


def _dy_w(g, W, M, K, N, mask=None):
    """dY W (M x K, reduced over W's N rows), zero where mask <= 0.  Wide layers over many rows go through the forward
    kernel with a transposed copy of W: gm_linear's 16-wave tile runs 13752 x 1744 x 1744 at 112 TFLOP/s where gm_gemm(0,1)
    reaches 96 (1744 x 1534: 112 vs 78), the copy costs 0.03 ms, and both walk the reduced dimension in ascending order
    from 0 -- the same bits wherever gm_gemm would not split the reduction, as on the tower shapes (tools/dx_ab.py)."""
    if M >= 4096 and N >= 1024 and K >= 1024:
        Wt = W.t().contiguous()
        out = torch.empty((M, K), dtype=torch.float32, device=g.device)
        L.call("gm_linear", I64(M), I64(K), I64(N), ptr(g), I64(N), ptr(Wt), I64(N), None, ptr(out), I64(K), I32(0), stream_ptr())
        if mask is not None:
            L.call("gm_relu_bwd", I64(out.numel()), ptr(out), ptr(mask), ptr(out), stream_ptr())
        return out
    return gemm(False, True, M, K, N, g, N, W, K, mask=mask)


def _linear_backward(x, W, g, needs):
    """(dx, dW, db) of y = x W^T + b for the gradient g of y (already masked by any ReLU)."""
    M, K = x.shape
    N = W.shape[0]
    dx = _dy_w(g, W, M, K, N) if needs[0] else None                               # dY W
    dW = gemm(True, True, N, K, M, g, N, x, K) if needs[1] else None              # dY^T X
    db = colsum(g) if needs[2] else None
    return dx, dW, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b, relu):
        x, W = _c(x), _c(W)
        require(x, torch.float32, "x")
        require(W, torch.float32, "W")
        M, K = x.shape
        N = W.shape[0]
        if W.shape[1] != K:
            raise ValueError(f"linear: x is {tuple(x.shape)}, W is {tuple(W.shape)}")
        y = torch.empty((M, N), dtype=torch.float32, device=x.device)
        L.call("gm_linear", I64(M), I64(N), I64(K), ptr(x), I64(K), ptr(W), I64(K), ptr(b), ptr(y), I64(N), I32(int(relu)),
               stream_ptr())
        ctx.relu = relu
        ctx.has_bias = b is not None
        ctx.save_for_backward(x, W, y if relu else None)
        return y

    @staticmethod
    def backward(ctx, g):
        x, W, y = ctx.saved_tensors
        g = _c(g)
        if ctx.relu:
            gm = torch.empty_like(g)
            L.call("gm_relu_bwd", I64(g.numel()), ptr(g), ptr(y), ptr(gm), stream_ptr())
            g = gm
        needs = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2])
        dx, dW, db = _linear_backward(x, W, g, needs)
        return dx, dW, db, None


class _Mlp2(torch.autograd.Function):
    """Linear -> ReLU -> Linear [-> ReLU] (mlp_in_X, mlp_out and the pair MLP, model/gnn.py:116-126,138-142,227-231) as one
    tape node, so that the backward applies the inner ReLU mask in the epilogue of the GEMM that produces the hidden
    gradient instead of in a pass of its own (the pair MLP's hidden gradient is batch x 128 floats: 1 GB per step)."""

    @staticmethod
    def forward(ctx, x, W1, b1, W2, b2, relu_out, onehot_sparse=None):
        x, W1, W2 = _c(x), _c(W1), _c(W2)
        require(x, torch.float32, "x")
        M, K = x.shape
        H, N = W1.shape[0], W2.shape[0]
        if W1.shape[1] != K or W2.shape[1] != H:
            raise ValueError(f"mlp2: x is {tuple(x.shape)}, W1 is {tuple(W1.shape)}, W2 is {tuple(W2.shape)}")
        if onehot_sparse is not None:
            # x is the one-hot attribute matrix (mlp_in_X): the first layer in the arithmetic of the fused tower call
            # (gm_onehot.hip), so that the tape's forward and gm_tower_forward give the same bits; the backward is unchanged
            y1 = ops.onehot_linear(ops.x_from_onehot(x), W1, b1, relu=True, sparse=bool(onehot_sparse))
        else:
            y1 = torch.empty((M, H), dtype=torch.float32, device=x.device)
            L.call("gm_linear", I64(M), I64(H), I64(K), ptr(x), I64(K), ptr(W1), I64(K), ptr(b1), ptr(y1), I64(H), I32(1),
                   stream_ptr())
        y2 = torch.empty((M, N), dtype=torch.float32, device=x.device)
        L.call("gm_linear", I64(M), I64(N), I64(H), ptr(y1), I64(H), ptr(W2), I64(H), ptr(b2), ptr(y2), I64(N), I32(int(relu_out)),
               stream_ptr())
        ctx.relu_out = relu_out
        ctx.has_bias = (b1 is not None, b2 is not None)
        ctx.save_for_backward(x, W1, W2, y1, y2 if relu_out else None)
        return y2

    @staticmethod
    def backward(ctx, g):
        x, W1, W2, y1, y2 = ctx.saved_tensors
        g = _c(g)
        if ctx.relu_out:
            gm = torch.empty_like(g)
            L.call("gm_relu_bwd", I64(g.numel()), ptr(g), ptr(y2), ptr(gm), stream_ptr())
            g = gm
        M, K = x.shape
        H, N = W1.shape[0], W2.shape[0]
        need = ctx.needs_input_grad
        dW2 = gemm(True, True, N, H, M, g, N, y1, H) if need[3] else None
        db2 = colsum(g) if ctx.has_bias[1] and need[4] else None
        want_db1 = ctx.has_bias[0] and need[2]
        ws_bytes = L.load().gm_mlp2_hidden_grad_workspace_bytes(I64(M), I64(H), I64(N))
        if ws_bytes >= 0:      # few outputs (the pair MLP): hidden gradient and its column sums in one pass over the batch
            g1 = torch.empty((M, H), dtype=torch.float32, device=g.device)
            db1 = torch.empty(H, dtype=torch.float32, device=g.device) if want_db1 else None
            ws = _scratch(ws_bytes, g.device) if want_db1 else None
            L.call("gm_mlp2_hidden_grad", I64(M), I64(H), I64(N), ptr(g), ptr(W2), I64(H), ptr(y1), ptr(g1), ptr(db1), ptr(ws),
                   I64(ws.numel() if ws is not None else 0), stream_ptr())
            dx, dW1, _ = _linear_backward(x, W1, g1, (need[0], need[1], False))
        else:
            g1 = _dy_w(g, W2, M, H, N, mask=y1)                            # (dY W2) where the hidden unit was active
            dx, dW1, db1 = _linear_backward(x, W1, g1, (need[0], need[1], want_db1))
        return dx, dW1, db1, dW2, db2, None, None


LAYERNORM_BWD_MAX = 1024        # gm_layernorm_bwd keeps a row's columns in registers; wider blocks use gm_layer_norm_bwd


class _UpdateBlock(torch.autograd.Function):
    """Linear -> ReLU -> LayerNorm of GNNLayer / MLPLayer (model/gnn.py:27-38)."""

    @staticmethod
    def forward(ctx, x, W, b, gamma, beta, eps):
        x, W = _c(x), _c(W)
        require(x, torch.float32, "x")
        M, K = x.shape
        N = W.shape[0]
        dev = x.device
        a = torch.empty((M, N), dtype=torch.float32, device=dev)
        L.call("gm_linear", I64(M), I64(N), I64(K), ptr(x), I64(K), ptr(W), I64(K), ptr(b), ptr(a), I64(N), I32(1), stream_ptr())
        y = torch.empty_like(a)
        mean = torch.empty(M, dtype=torch.float32, device=dev)
        rstd = torch.empty(M, dtype=torch.float32, device=dev)
        L.call("gm_layernorm_fwd", I64(M), I64(N), ptr(a), I64(N), ptr(gamma), ptr(beta), F32(eps), ptr(y), I64(N), ptr(mean),
               ptr(rstd), stream_ptr())
        ctx.save_for_backward(x, W, a, mean, rstd, gamma)
        return y

    @staticmethod
    def backward(ctx, g):
        x, W, a, mean, rstd, gamma = ctx.saved_tensors
        g = _c(g)
        M, N = a.shape
        dev = a.device
        da = torch.empty_like(a)
        dgb = torch.empty((2, N), dtype=torch.float32, device=dev)
        if N > LAYERNORM_BWD_MAX:
            _layer_norm_bwd(g, a, M, N, 0, mean.data_ptr(), rstd.data_ptr(), gamma, 0, da, dgb[0], dgb[1])
            L.call("gm_relu_bwd", I64(a.numel()), ptr(da), ptr(a), ptr(da), stream_ptr())
            dx, dW, db = _linear_backward(x, W, da, (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]))
            return dx, dW, db, dgb[0], dgb[1], None
        need = L.load().gm_layernorm_bwd_workspace_bytes(I64(M), I64(N))
        ws = _scratch(need, dev)
        L.call("gm_layernorm_bwd", I64(M), I64(N), ptr(g), I64(N), ptr(a), I64(N), ptr(mean), ptr(rstd), ptr(gamma), I32(1),
               ptr(da), I64(N), ptr(dgb), C_void(dgb, N), ptr(ws), I64(ws.numel()), stream_ptr())
        dx, dW, db = _linear_backward(x, W, da, (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[2]))
        return dx, dW, db, dgb[0], dgb[1], None


class _SpmmMean(torch.autograd.Function):
    @staticmethod
    def forward(ctx, H, adj):
        H = _c(H)
        require(H, torch.float32, "H")
        n, d = H.shape
        out = torch.empty_like(H)
        L.call("gm_spmm_mean", I64(n), ptr(adj.rowptr), ptr(adj.colidx), ptr(H), I64(d), I64(d), ptr(out), I64(d), stream_ptr())
        ctx.adj = adj
        return out

    @staticmethod
    def backward(ctx, g):
        g = _c(g)
        n, d = g.shape
        adj = ctx.adj
        out = torch.empty_like(g)
        L.call("gm_spmm_mean_bwd", I64(n), ptr(adj.rowptr), ptr(adj.colidx), ptr(g), I64(d), I64(d), ptr(out), I64(d),
               stream_ptr())
        return out, None


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, idx32):
        weight = _c(weight)
        require(weight, torch.float32, "emb.weight")
        require(idx32, torch.int32, "idx")
        n = idx32.numel()
        Cn, w = weight.shape
        ops.check_index_range(idx32, Cn, "Y")
        out = torch.empty((n, w), dtype=torch.float32, device=weight.device)
        L.call("gm_embedding_fwd", I64(n), I32(Cn), I32(w), ptr(idx32), ptr(weight), I64(w), ptr(out), I64(w), stream_ptr())
        ctx.save_for_backward(idx32)
        ctx.shape = (Cn, w)
        return out

    @staticmethod
    def backward(ctx, g):
        (idx32,) = ctx.saved_tensors
        g = _c(g)
        Cn, w = ctx.shape
        dW = torch.empty((Cn, w), dtype=torch.float32, device=g.device)
        ws = _scratch(L.load().gm_embedding_bwd_workspace_bytes(I64(idx32.numel()), I32(Cn), I32(w)), g.device)
        L.call("gm_embedding_bwd", I64(idx32.numel()), I32(Cn), I32(w), ptr(idx32), ptr(g), I64(w), ptr(dW), I64(w), ptr(ws),
               I64(ws.numel()), stream_ptr())
        return dW, None


class _HadamardGather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, src, dst):
        h = _c(h)
        require(h, torch.float32, "h")
        src, dst = _c(src), _c(dst)
        require(src, torch.int64, "src")
        require(dst, torch.int64, "dst")
        B, d = src.numel(), h.shape[1]
        ops.check_index_range(src, h.shape[0], "src")
        ops.check_index_range(dst, h.shape[0], "dst")
        out = torch.empty((B, d), dtype=torch.float32, device=h.device)
        L.call("gm_hadamard_gather", I64(B), I64(d), ptr(src), ptr(dst), ptr(h), I64(d), ptr(out), I64(d), stream_ptr())
        ctx.save_for_backward(h, src, dst)
        return out

    @staticmethod
    def backward(ctx, g):
        h, src, dst = ctx.saved_tensors
        g = _c(g)
        n, d = h.shape
        B = src.numel()
        # group the 2B (pair, role) entries by node: index plumbing (a stable sort of the ids), then one kernel
        keys = torch.cat([src, dst])
        # node ids fit 16 (or 32) bits: the radix sort then makes 2 (4) passes over the 2B keys instead of 8
        narrow = keys.to(torch.int16) if n <= 32767 else keys.to(torch.int32) if n <= 2**31 - 1 else keys
        order = torch.argsort(narrow, stable=True)
        counts = torch.bincount(keys, minlength=n)
        segptr = torch.zeros(n + 1, dtype=torch.int64, device=h.device)
        segptr[1:] = torch.cumsum(counts, 0)
        dh = torch.empty_like(h)
        L.call("gm_hadamard_gather_bwd", I64(n), I64(B), I64(d), ptr(src), ptr(dst), ptr(segptr), ptr(order), ptr(h), I64(d),
               ptr(g), I64(d), ptr(dh), I64(d), stream_ptr())
        return dh, None, None


class _SoftmaxCE2(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target_u8):
        logits = _c(logits)
        require(logits, torch.float32, "logits")
        require(target_u8, torch.uint8, "target")
        total = target_u8.numel()
        if logits.numel() != 2 * total:
            raise ValueError(f"softmax_ce2: {logits.numel()} logits for {total} targets")
        dev = logits.device
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        dl = torch.empty_like(logits) if ctx.needs_input_grad[0] else None
        ws = _scratch(L.load().gm_softmax_ce2_workspace_bytes(), dev, slot=1)
        L.call("gm_softmax_ce2", I64(total), ptr(logits), ptr(target_u8), ptr(loss), ptr(dl), ptr(ws), I64(ws.numel()),
               stream_ptr())
        ctx.save_for_backward(dl)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        (dl,) = ctx.saved_tensors
        return dl * g, None


class _CE2Diff(torch.autograd.Function):
    """Two-class cross entropy from the logit difference d = l1 - l0 (gm_ce2_diff)."""

    @staticmethod
    def forward(ctx, diff, target_u8):
        diff = _c(diff)
        require(diff, torch.float32, "diff")
        require(target_u8, torch.uint8, "target")
        total = target_u8.numel()
        if diff.numel() != total:
            raise ValueError(f"ce2_diff: {diff.numel()} differences for {total} targets")
        dev = diff.device
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        dd = torch.empty_like(diff) if ctx.needs_input_grad[0] else None
        ws = _scratch(L.load().gm_softmax_ce2_workspace_bytes(), dev, slot=1)
        L.call("gm_ce2_diff", I64(total), ptr(diff), ptr(target_u8), ptr(loss), ptr(dd), ptr(ws), I64(ws.numel()), stream_ptr())
        ctx.save_for_backward(dd)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        (dd,) = ctx.saved_tensors
        return dd * g, None


class _HeadDiff(torch.autograd.Function):
    """(Wd, bd) = (W[1::2] - W[0::2], b[1::2] - b[0::2]) of a two-class head (gm_head_diff_prepare); the gradient goes back
    as dW[1::2] = dWd, dW[0::2] = -dWd (gm_head_diff_bwd)."""

    @staticmethod
    def forward(ctx, W, b):
        W, b = _c(W), _c(b)
        Wd, bd = ops.head_diff(W, b)
        ctx.shape = tuple(W.shape)
        return Wd, bd

    @staticmethod
    def backward(ctx, gWd, gbd):
        F2, Hc = ctx.shape
        if gWd is None:
            gWd = torch.zeros((F2 // 2, Hc), dtype=torch.float32, device=gbd.device)
        gWd = _c(gWd)
        gbd = _c(gbd) if gbd is not None else None
        dW = torch.empty((F2, Hc), dtype=torch.float32, device=gWd.device)
        db = torch.empty(F2, dtype=torch.float32, device=gWd.device) if gbd is not None else None
        L.call("gm_head_diff_bwd", I64(F2 // 2), I64(Hc), ptr(gWd), ptr(gbd), ptr(dW), ptr(db), stream_ptr())
        return dW, db


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, call):
        x = _c(x)
        out = torch.empty_like(x)
        L.call("gm_dropout", I64(x.numel()), ptr(x), F32(p), U64(seed), U32(call), ptr(out), stream_ptr())
        ctx.args = (p, seed, call)
        return out

    @staticmethod
    def backward(ctx, g):
        g = _c(g)
        p, seed, call = ctx.args
        out = torch.empty_like(g)
        L.call("gm_dropout", I64(g.numel()), ptr(g), F32(p), U64(seed), U32(call), ptr(out), stream_ptr())
        return out, None, None, None


def linear(x, W, b=None, relu=False):
    return _Linear.apply(x, W, b, relu)


def mlp2(x, W1, b1, W2, b2, relu_out=False, onehot_sparse=None):
    """onehot_sparse: None = a general input; False / True = x is the towers' one-hot attribute matrix and the first layer
    runs in the dense / sparse one-hot form (include/graphmaker_hip.h, gm_onehot_linear)."""
    return _Mlp2.apply(x, W1, b1, W2, b2, relu_out, onehot_sparse)


def update_block(x, W, b, gamma, beta, eps=1e-5):
    return _UpdateBlock.apply(x, W, b, gamma, beta, eps)


def spmm_mean(adj, H):
    return _SpmmMean.apply(H, adj)


def embedding(weight, idx32):
    return _Embedding.apply(weight, idx32)


def hadamard_gather(h, src, dst):
    return _HadamardGather.apply(h, src, dst)


def softmax_ce2(logits, target_u8):
    return _SoftmaxCE2.apply(logits, target_u8)


def ce2_diff(diff, target_u8):
    return _CE2Diff.apply(diff, target_u8)


def head_diff(W, b):
    return _HeadDiff.apply(W, b)


class DropoutState:
    """Seed and call counter of the dropout masks of one model (a fresh mask per application, reproducible per seed)."""

    def __init__(self, seed=0):
        self.seed, self.calls = int(seed) & 0xFFFFFFFFFFFFFFFF, 0

    def next(self):
        self.calls = (self.calls + 1) & 0xFFFFFFFF
        return self.seed, self.calls


def dropout(x, p, state):
    if p <= 0.0:
        return x
    seed, call = state.next()
    return _Dropout.apply(x, float(p), seed, call)


# ------------------------------------------------------------------ wider models and fine-tuning
# A small call costs what its Python costs (the kernels of a short sequence take a few microseconds, the autograd engine's
# round trip some 30): contiguous tensors are used as they are, without a view, and backward passes get their sizes as numbers.
def _gradient(fn):
    """A backward pass without a second derivative: an error for who differentiates the gradient (create_graph), and no wrapper
    around the call otherwise."""
    checked = once_differentiable(fn)

    def backward(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


def _on_gpu(t, what):
    if not t.is_cuda:
        raise L.GraphMakerHipError(f"{what}: graphmaker_amd runs on a ROCm device only (tensor is on {t.device})")


def _same_device(t, what, device):
    if t.device != device:
        raise ValueError(f"{what}: on {t.device}, expected {device}")
    return t


def _row_dtype(t, what):
    code = L.DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows(t, width):
    """(tensor, leading dimension) of t as rows of `width` elements at its address; a copy only where its strides need one."""
    if t.is_contiguous():
        return t, width
    t = t.reshape(-1, width)
    if t.shape[0] == 0 or (t.shape[0] == 1 and (width == 1 or t.stride(1) == 1)):
        return t, width
    if (width > 1 and t.stride(1) != 1) or t.stride(0) < width:
        t = t.contiguous()
    return t, t.stride(0)


def _index(t, what, device):
    """(contiguous tensor, 1 if int64) of an index argument."""
    i64 = t.dtype == torch.int64
    if not i64 and t.dtype != torch.int32:
        raise TypeError(f"{what}: expected int32 or int64, got {t.dtype}")
    return _c(_same_device(t, what, device)), int(i64)


def _at(t):
    return t.data_ptr() if t is not None else None


def _token_embedding_fwd(weight, tokens, args):
    n, C, w, i64, code, scale, _, _ = args
    table, ldw = _rows(weight, w)
    out = torch.empty((*tokens.shape, w), dtype=weight.dtype, device=weight.device)
    L.launch("gm_token_embedding_fwd", weight.device, n, C, w, tokens.data_ptr(), i64, table.data_ptr(), ldw, code, scale, out.data_ptr(), w)
    return out


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, args):
        ctx.save_for_backward(tokens)
        ctx.args = args
        return _token_embedding_fwd(weight, tokens, args)

    @_gradient
    def backward(ctx, g):
        (tokens,) = ctx.saved_tensors
        n, C, w, i64, code, scale, padding, need = ctx.args
        dev = g.device
        g, ldg = _rows(g, w)
        dW = torch.empty((C, w), dtype=g.dtype, device=dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        L.launch("gm_token_embedding_bwd", dev, n, C, w, tokens.data_ptr(), i64, padding, g.data_ptr(), ldg, code, scale, dW.data_ptr(), w,
                 ws.data_ptr(), need)
        return dW, None, None


def token_embedding(weight, tokens, scale=1.0, padding_idx=None):
    """scale * weight[tokens], shape tokens.shape + (w,), in weight's type (float32, bfloat16, float16).  tokens: int32 or int64
    of any shape.  The gradient sums each row's tokens in ascending position (no atomics: the same bits on every run) and
    leaves row padding_idx zero, as nn.Embedding does.  Tokens are not read on the host: one outside [0, C) gives a row of
    NaN and adds to no gradient; ops.check_index_range(tokens, C, "tokens") is the check that raises."""
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"token_embedding: weight must be (C, w) with C, w > 0, got {tuple(weight.shape)}")
    code = _row_dtype(weight, "weight")
    tokens, i64 = _index(tokens, "tokens", weight.device)
    C, w = weight.shape
    if padding_idx is None:
        padding = -1
    else:
        if not -C <= padding_idx < C:
            raise ValueError(f"token_embedding: padding_idx {padding_idx} is outside the {C} rows of weight")
        padding = int(padding_idx) % C
    _on_gpu(weight, "weight")
    n = tokens.numel()
    if weight.requires_grad and torch.is_grad_enabled():
        need = L.function("gm_token_embedding_bwd_workspace_bytes")(n, C, w)
        return _TokenEmbedding.apply(weight, tokens, (n, C, w, i64, code, float(scale), padding, need))
    return _token_embedding_fwd(weight, tokens, (n, C, w, i64, code, float(scale), padding, 0))


def _layer_norm_fwd(x, gamma, beta, args, stats):
    M, N, code, wcode, eps = args
    dev = x.device
    rows, ldx = _rows(x, N)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    st = torch.empty(2 * M, dtype=torch.float32, device=dev) if stats else None
    at = _at(st)
    L.launch("gm_layer_norm_fwd", dev, M, N, rows.data_ptr(), ldx, code, _at(gamma), _at(beta), wcode, eps, y.data_ptr(), N, at,
             at + 4 * M if at else at)
    return y, rows, st


def _layer_norm_bwd(g, rows, M, N, code, mean, rstd, gamma, wcode, dx, dgamma, dbeta):
    """gm_layer_norm_bwd over the M rows of N of x; mean, rstd: addresses; dx, dgamma, dbeta: outputs or None."""
    dev = rows.device
    rows, ldx = _rows(rows, N)
    g, ldg = _rows(g, N)
    need = L.function("gm_layer_norm_bwd_workspace_bytes")(M, N) if dgamma is not None or dbeta is not None else 0
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    L.launch("gm_layer_norm_bwd", dev, M, N, g.data_ptr(), ldg, rows.data_ptr(), ldx, code, mean, rstd, _at(gamma), wcode, _at(dx), N,
             _at(dgamma), _at(dbeta), _at(ws), need)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, args):
        y, rows, st = _layer_norm_fwd(x, gamma, beta, args, True)
        ctx.save_for_backward(rows, st, gamma)
        ctx.args = args
        ctx.shape = x.shape
        ctx.weight_dtypes = (gamma.dtype if gamma is not None else None, beta.dtype if beta is not None else None)
        return y

    @_gradient
    def backward(ctx, g):
        rows, st, gamma = ctx.saved_tensors
        M, N, code, wcode, _ = ctx.args
        dev, need, types = g.device, ctx.needs_input_grad, ctx.weight_dtypes
        dx = torch.empty(ctx.shape, dtype=g.dtype, device=dev) if need[0] else None
        dgamma = torch.empty(N, dtype=types[0], device=dev) if need[1] else None
        dbeta = torch.empty(N, dtype=types[1], device=dev) if need[2] else None
        at = st.data_ptr()
        _layer_norm_bwd(g, rows, M, N, code, at, at + 4 * M, gamma, wcode, dx, dgamma, dbeta)
        return dx, dgamma, dbeta, None


def layer_norm(x, gamma=None, beta=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * gamma + beta over the last dimension, of any width, in x's type (float32, bfloat16,
    float16).  gamma and beta (N,): x's type or float32, both the same; None: 1 and 0.  Statistics are float32 about the mean,
    the variance that of the differences from it."""
    N = x.shape[-1] if x.dim() else 0
    if N == 0:
        raise ValueError(f"layer_norm: x must have a last dimension of at least 1, got {tuple(x.shape)}")
    code = _row_dtype(x, "x")
    wcode, records = code, x.requires_grad
    for t, what in ((gamma, "gamma"), (beta, "beta")):
        if t is None:
            continue
        if t.dim() != 1 or t.numel() != N:
            raise ValueError(f"layer_norm: {what} is {tuple(t.shape)}, x's rows have {N} columns")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"layer_norm: {what} is {t.dtype}, expected {x.dtype} or float32")
        _same_device(t, what, x.device)
        wcode = L.DTYPES[t.dtype]
        records = records or t.requires_grad
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        raise TypeError(f"layer_norm: gamma is {gamma.dtype} and beta is {beta.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    _on_gpu(x, "x")
    gamma, beta = (t if t is None else _c(t) for t in (gamma, beta))
    args = (x.numel() // N, N, code, wcode, float(eps))
    if records and torch.is_grad_enabled():
        return _LayerNorm.apply(x, gamma, beta, args)
    return _layer_norm_fwd(x, gamma, beta, args, False)[0]


def _class_log_prob_fwd(logits, classes, args, stats):
    M, V, code, i64, ignore_index = args
    dev = logits.device
    rows, ldx = _rows(logits, V)
    lp = torch.empty(classes.shape, dtype=torch.float32, device=dev)
    floats = L.function("gm_class_log_prob_stats_floats")(M, V, code) if stats else 0
    st = torch.empty(floats, dtype=torch.float32, device=dev) if floats else None
    need = L.function("gm_class_log_prob_workspace_bytes")(M, V, code)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    L.launch("gm_class_log_prob_fwd", dev, M, V, rows.data_ptr(), ldx, code, classes.data_ptr(), i64, ignore_index, lp.data_ptr(), _at(st),
             _at(ws), need)
    return lp, rows, ldx, st


class _ClassLogProb(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, classes, args):
        lp, rows, ctx.ldx, st = _class_log_prob_fwd(logits, classes, args, True)
        ctx.save_for_backward(rows, classes, st)
        ctx.args = args
        ctx.shape = logits.shape
        return lp

    @_gradient
    def backward(ctx, g):
        rows, classes, st = ctx.saved_tensors
        M, V, code, i64, ignore_index = ctx.args
        g = _c(g)
        dx = torch.empty(ctx.shape, dtype=rows.dtype, device=g.device)
        L.launch("gm_class_log_prob_bwd", g.device, M, V, g.data_ptr(), rows.data_ptr(), ctx.ldx, code, classes.data_ptr(), i64, ignore_index,
                 _at(st), dx.data_ptr(), V)
        return dx, None, None


def class_log_prob(logits, classes, ignore_index=-100):
    """log softmax(logits)[classes] over the last dimension: float32 of shape classes.shape = logits.shape[:-1]; logits float32,
    bfloat16 or float16, classes int32 or int64.  A row whose class is ignore_index has log-probability 0 and a zero gradient,
    whatever its logits hold; any other class outside [0, V) gives NaN in both (classes are not read on the host).  A row
    whose upstream gradient is exactly 0 gets a zero gradient too."""
    V = logits.shape[-1] if logits.dim() else 0
    if V == 0:
        raise ValueError(f"class_log_prob: logits must have a last dimension of at least 1, got {tuple(logits.shape)}")
    if classes.shape != logits.shape[:-1]:
        raise ValueError(f"class_log_prob: classes is {tuple(classes.shape)}, logits is {tuple(logits.shape)}")
    code = _row_dtype(logits, "logits")
    classes, i64 = _index(classes, "classes", logits.device)
    _on_gpu(logits, "logits")
    args = (classes.numel(), V, code, i64, int(ignore_index))
    if logits.requires_grad and torch.is_grad_enabled():
        return _ClassLogProb.apply(logits, classes, args)
    return _class_log_prob_fwd(logits, classes, args, False)[0]


def _items(t, what, like=None):
    """A float32 per-item argument; with `like`, one of its shape and device that takes no gradient."""
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: expected float32, got {t.dtype}")
    if like is not None:
        if t.shape != like.shape:
            raise ValueError(f"{what} is {tuple(t.shape)}, log_prob is {tuple(like.shape)}")
        _constant(t, what)
        _same_device(t, what, like.device)
    return _c(t)


def _constant(t, what):
    if t.requires_grad:
        raise ValueError(f"{what} is a constant of the loss and gets no gradient: pass {what}.detach()")


def _mask(mask, like):
    if mask is None:
        return None
    if mask.dtype != torch.bool and mask.dtype != torch.uint8:
        raise TypeError(f"mask: expected bool or uint8, got {mask.dtype}")
    if mask.shape != like.shape:
        raise ValueError(f"mask is {tuple(mask.shape)}, log_prob is {tuple(like.shape)}")
    return _c(_same_device(mask, "mask", like.device))


def _offsets(offsets, device):
    if offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError(f"offsets: expected the S + 1 borders of S > 0 sequences, got {tuple(offsets.shape)}")
    return _index(offsets, "offsets", device)


def _sequence_buffer(M, S, slopes, dev):
    """(buffer, addresses of the S weights, `slopes` slopes and the workspace in it, workspace bytes).  What a loss keeps for its
    backward pass and what it works in share one allocation."""
    need = L.function("gm_sequence_loss_workspace_bytes")(M, S)
    head = (4 * (S + slopes) + 15) // 16 * 16
    buf = torch.empty(head + need, dtype=torch.uint8, device=dev)
    at = buf.data_ptr()
    return buf, at, at + 4 * S if slopes else None, at + head, need


def _sequence_loss_bwd(g, buf, M, S, has_slope, mask, offsets, i64, shape):
    out = torch.empty(shape, dtype=torch.float32, device=g.device)
    at = buf.data_ptr()
    L.launch("gm_sequence_loss_bwd", g.device, M, S, at + 4 * S if has_slope else None, _at(mask), _at(offsets), i64, at, g.data_ptr(),
             out.data_ptr())
    return out


def _policy_loss_fwd(lp, old, adv, ref, mask, offsets, args, grad):
    M, S, i64, clip_low, clip_high, kl_coef, by_sequence = args
    dev = lp.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    stats = torch.empty(4, dtype=torch.float32, device=dev)
    buf, weight, slope, ws, need = _sequence_buffer(M, S, M if grad else 0, dev)
    L.launch("gm_policy_loss_fwd", dev, M, S, lp.data_ptr(), old.data_ptr(), adv.data_ptr(), _at(ref), _at(mask), _at(offsets), i64, clip_low,
             clip_high, kl_coef, by_sequence, loss.data_ptr(), stats.data_ptr(), slope, weight, ws, need)
    return loss, stats, buf


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lp, old, adv, ref, mask, offsets, args):
        loss, stats, buf = _policy_loss_fwd(lp, old, adv, ref, mask, offsets, args, True)
        ctx.save_for_backward(buf, mask, offsets)
        ctx.args = args
        ctx.shape = lp.shape
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @_gradient
    def backward(ctx, g, _stats):
        if g is None:
            return (None,) * 7
        buf, mask, offsets = ctx.saved_tensors
        M, S, i64 = ctx.args[:3]
        return _sequence_loss_bwd(g, buf, M, S, M > 0, mask, offsets, i64, ctx.shape), None, None, None, None, None, None


def policy_loss(log_prob, old_log_prob, advantage, *, offsets=None, mask=None, ref_log_prob=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, reduction="token"):
    """Clipped policy loss of the items' log-probabilities (float32, any shape; see class_log_prob) against those under the
    model that drew them:  r = exp(log_prob - old_log_prob),  -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
    + kl_coef * (exp(q) - q - 1),  q = ref_log_prob - log_prob.

    offsets: S + 1 non-decreasing borders (int32 / int64) of consecutive sequences of items; `advantage` then has one value a
    sequence, without offsets one an item.  mask: bool / uint8.  An item outside every sequence or masked off counts nowhere,
    whatever its values, and gets a zero gradient.  reduction: "token" averages over the live items, "sequence" over each
    sequence's and then over the sequences that have one; without any live item the loss is 0.  old_log_prob, advantage and
    ref_log_prob are constants.

    Returns (loss, stats), stats = [mean surrogate, mean KL, share of clipped items, live items] without a gradient."""
    lp = _items(log_prob, "log_prob")
    old = _items(old_log_prob, "old_log_prob", log_prob)
    ref = _items(ref_log_prob, "ref_log_prob", log_prob) if ref_log_prob is not None else None
    mask = _mask(mask, log_prob)
    i64, S = 0, 1
    if offsets is None:
        adv = _items(advantage, "advantage", log_prob)
    else:
        offsets, i64 = _offsets(offsets, log_prob.device)
        S = offsets.numel() - 1
        adv = _items(advantage, "advantage")
        _same_device(adv, "advantage", log_prob.device)
        _constant(advantage, "advantage")
        if advantage.dim() != 1 or advantage.numel() != S:
            raise ValueError(f"advantage is {tuple(advantage.shape)}, offsets border {S} sequences")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction: expected 'token' or 'sequence', got {reduction!r}")
    if reduction == "sequence" and offsets is None:
        raise ValueError("reduction 'sequence' needs offsets")
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError(f"clip range: 0 <= clip_low <= 1 and 0 <= clip_high, got {clip_low}, {clip_high}")
    if kl_coef != 0.0 and ref is None:
        raise ValueError("kl_coef needs ref_log_prob")
    if kl_coef - kl_coef != 0.0:
        raise ValueError(f"kl_coef must be finite, got {kl_coef}")
    _on_gpu(log_prob, "log_prob")
    args = (lp.numel(), S, i64, float(clip_low), float(clip_high), float(kl_coef), int(reduction == "sequence"))
    if log_prob.requires_grad and torch.is_grad_enabled():
        return _PolicyLoss.apply(lp, old, adv, ref, mask, offsets, args)
    return _policy_loss_fwd(lp, old, adv, ref, mask, offsets, args, False)[:2]


def _preference_loss_fwd(lp, ref, mask, offsets, args):
    M, S, i64, beta, smoothing, average = args
    dev = lp.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rewards = torch.empty(S, dtype=torch.float32, device=dev)
    buf, weight, _, ws, need = _sequence_buffer(M, S, 0, dev)
    L.launch("gm_preference_loss_fwd", dev, M, S // 2, lp.data_ptr(), ref.data_ptr(), _at(mask), offsets.data_ptr(), i64, beta, smoothing, average,
             loss.data_ptr(), rewards.data_ptr(), weight, ws, need)
    return loss, rewards, buf


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lp, ref, mask, offsets, args):
        loss, rewards, buf = _preference_loss_fwd(lp, ref, mask, offsets, args)
        ctx.save_for_backward(buf, mask, offsets)
        ctx.args = args
        ctx.shape = lp.shape
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @_gradient
    def backward(ctx, g, _rewards):
        if g is None:
            return (None,) * 5
        buf, mask, offsets = ctx.saved_tensors
        M, S, i64 = ctx.args[:3]
        return _sequence_loss_bwd(g, buf, M, S, False, mask, offsets, i64, ctx.shape), None, None, None, None


def preference_loss(log_prob, ref_log_prob, offsets, *, mask=None, beta=0.1, label_smoothing=0.0, average=False):
    """Loss of P pairs of sequences from the items' log-probabilities under the trained and a reference model (float32):
    sequence 2p of the 2P that the 2P + 1 `offsets` border is preferred over sequence 2p + 1.  h = sum (average=True: mean) over
    a sequence's live items of log_prob - ref_log_prob,  z = beta (h_2p - h_2p+1),
    mean over pairs of -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z).

    mask, items outside every sequence: as in policy_loss.  A sequence without a live item has h = 0.
    Returns (loss, rewards), rewards = beta h of the 2P sequences, without a gradient."""
    lp = _items(log_prob, "log_prob")
    ref = _items(ref_log_prob, "ref_log_prob", log_prob)
    mask = _mask(mask, log_prob)
    offsets, i64 = _offsets(offsets, log_prob.device)
    S = offsets.numel() - 1
    if S % 2:
        raise ValueError(f"offsets border {S} sequences: an even number makes pairs")
    if not 0.0 < beta < float("inf") or not 0.0 <= label_smoothing <= 0.5:
        raise ValueError(f"0 < beta and 0 <= label_smoothing <= 0.5, got {beta}, {label_smoothing}")
    _on_gpu(log_prob, "log_prob")
    args = (lp.numel(), S, i64, float(beta), float(label_smoothing), int(bool(average)))
    if log_prob.requires_grad and torch.is_grad_enabled():
        return _PreferenceLoss.apply(lp, ref, mask, offsets, args)
    return _preference_loss_fwd(lp, ref, mask, offsets, args)[:2]
