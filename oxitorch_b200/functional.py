"""Device-side mirror of oxitorch's ``F.*`` layer functions.

Same names, argument meaning and error behaviour as
``python/oxitorch/nn/functional.py`` for the memory-bound layers; each call is
one fused CUDA kernel through liboxicuda.so, and its VJP is one fused kernel
(plus a deterministic column-sum finisher for weight gradients).  Tensors are
torch CUDA float32 tensors: torch supplies device memory, the stream and the
autograd graph bookkeeping (``torch.autograd.Function``); all arithmetic on
the path is ours.

The last parts of the file, the layers of a recurrent draft model and those of a
selective state space model with its policy loss, have no counterpart in the
reference and take bfloat16 activations too.

``grad_mode`` selects the backward semantics of the norms:
``"ref"`` (default) reproduces the reference graph, where ``rsqrt`` is
detached (crates/oxi-bindings/src/lib.rs:682-697); ``"exact"`` is the full
mathematical gradient.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

import ctypes

from . import _native as N

_MODES = {"ref": N.GRAD_REF, "exact": N.GRAD_EXACT}


def _stream() -> int:
    # torch.cuda.current_stream().cuda_stream without the Stream object around it
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _require_cuda_f32(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if not t.is_cuda:
        raise ValueError(f"invalid argument: {name} must live on a CUDA device "
                         "(oxitorch_b200 has no CPU path)")
    if t.dtype != torch.float32:
        raise ValueError(f"invalid argument: {name} must be float32, got {t.dtype}")


def _rows_cols(x):
    if x.dim() == 0:
        raise ValueError("invalid argument: dim -1 out of range for 0-D tensor")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    return rows, cols


def dense(t):
    """t itself when it is dense row-major, else a dense copy made on the
    device by oxc_contiguous (the reference's Tensor::contiguous,
    crates/oxi-tensor/src/lib.rs:220-240): strided and transposed views reach
    the fused row kernels through one copy kernel of this library."""
    if t.is_contiguous():
        return t
    _require_cuda_f32("tensor", t)
    out = torch.empty(t.shape, dtype=torch.float32, device=t.device)
    N.check(N.load().oxc_contiguous(ctypes.byref(N.make_view(t)), ctypes.byref(N.make_view(out)),
                                    _stream()), "contiguous")
    return out


def _row_major(name, t):
    """The fused row kernels read dense rows: a strided view is copied first
    (the reference's compositions accept any view and produce dense results)."""
    return dense(t)


def _vector(name, t, cols):
    """A [cols] parameter; a broadcast view with zero row strides is accepted
    and read through its first row (no copy)."""
    if t.dim() >= 1 and t.shape[-1] == cols and all(s == 0 for s in t.stride()[:-1]):
        t = t.reshape(-1)[:cols] if t.dim() == 1 else t.select(0, 0) if t.dim() == 2 else t
    if t.dim() != 1 or t.shape[0] != cols:
        raise ValueError(f"shape mismatch: {list(t.shape)} vs [{cols}]")
    if t.stride(0) != 1:
        raise ValueError(f"invalid argument: {name} must be contiguous")
    return t


def _workspace(nbytes, device):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


# ---- RMSNorm ---------------------------------------------------------------------

def rms_norm_fwd(x, weight, eps=1e-6):
    """Returns (y, rstd) for x [..., cols]."""
    _require_cuda_f32("x", x)
    _require_cuda_f32("weight", weight)
    x = _row_major("x", x)
    rows, cols = _rows_cols(x)
    weight = _vector("weight", weight, cols)
    y = torch.empty_like(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    L = N.load()
    N.check(L.oxc_rms_norm_fwd(x.data_ptr(), weight.data_ptr(), y.data_ptr(), rstd.data_ptr(),
                               rows, cols, float(eps), _stream()), "rms_norm")
    return y, rstd


def rms_norm_bwd(x, weight, rstd, dy, grad_mode="ref"):
    """Returns (dx, dweight)."""
    x = _row_major("x", x)
    rows, cols = _rows_cols(x)
    weight = _vector("weight", weight, cols)
    dy = _row_major("dy", dy)
    dx = torch.empty_like(x)
    dw = torch.empty(cols, dtype=torch.float32, device=x.device)
    L = N.load()
    ws_bytes = L.oxc_rms_norm_bwd_workspace_size(rows, cols)
    ws = _workspace(ws_bytes, x.device)
    N.check(L.oxc_rms_norm_bwd(x.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dy.data_ptr(),
                               dx.data_ptr(), dw.data_ptr(), rows, cols, _MODES[grad_mode],
                               ws.data_ptr(), ws.numel(), _stream()), "rms_norm backward")
    return dx, dw


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, grad_mode):
        x = dense(x)
        y, rstd = rms_norm_fwd(x, weight, eps)
        ctx.save_for_backward(x, weight, rstd)
        ctx.grad_mode = grad_mode
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, rstd = ctx.saved_tensors
        dx, dw = rms_norm_bwd(x, weight, rstd, dense(dy), ctx.grad_mode)
        return dx, dw.reshape(weight.shape), None, None


def rms_norm(x, weight, eps=1e-6, grad_mode="ref"):
    """F.rms_norm (python/oxitorch/nn/functional.py:236-240): x / rms(x) * weight."""
    return _RMSNorm.apply(x, weight, eps, grad_mode)


# ---- LayerNorm (+ GELU) --------------------------------------------------------------

def layer_norm_fwd(x, weight, bias, eps=1e-5, act=N.ACT_NONE):
    """Returns (y, mean, rstd); y = act(layer_norm(x))."""
    _require_cuda_f32("x", x)
    _require_cuda_f32("weight", weight)
    _require_cuda_f32("bias", bias)
    x = _row_major("x", x)
    rows, cols = _rows_cols(x)
    weight = _vector("weight", weight, cols)
    bias = _vector("bias", bias, cols)
    y = torch.empty_like(x)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    L = N.load()
    N.check(L.oxc_layer_norm_fwd(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(),
                                 mean.data_ptr(), rstd.data_ptr(), rows, cols, float(eps), act,
                                 _stream()), "layer_norm")
    return y, mean, rstd


def layer_norm_bwd(x, weight, bias, mean, rstd, dy, act=N.ACT_NONE, grad_mode="ref"):
    """Returns (dx, dweight, dbias)."""
    x = _row_major("x", x)
    rows, cols = _rows_cols(x)
    weight = _vector("weight", weight, cols)
    bias = _vector("bias", bias, cols)
    dy = _row_major("dy", dy)
    dx = torch.empty_like(x)
    dw = torch.empty(cols, dtype=torch.float32, device=x.device)
    db = torch.empty_like(dw)
    L = N.load()
    ws = _workspace(L.oxc_layer_norm_bwd_workspace_size(rows, cols), x.device)
    N.check(L.oxc_layer_norm_bwd(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), mean.data_ptr(),
                                 rstd.data_ptr(), dy.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                                 db.data_ptr(), rows, cols, act, _MODES[grad_mode], ws.data_ptr(),
                                 ws.numel(), _stream()), "layer_norm backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, act, grad_mode):
        x = dense(x)
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps, act)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.act, ctx.grad_mode = act, grad_mode
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(x, weight, bias, mean, rstd, dense(dy), ctx.act,
                                    ctx.grad_mode)
        return dx, dw.reshape(weight.shape), db.reshape(bias.shape), None, None, None


def layer_norm(x, weight, bias, eps=1e-5, grad_mode="ref"):
    """F.layer_norm (functional.py:227-233) over the last dim with affine weight/bias."""
    return _LayerNorm.apply(x, weight, bias, eps, N.ACT_NONE, grad_mode)


def layer_norm_gelu(x, weight, bias, eps=1e-5, grad_mode="ref"):
    """F.gelu(F.layer_norm(x, weight, bias, eps)) as one fused kernel each way
    (functional.py:227-233 then 194-199)."""
    return _LayerNorm.apply(x, weight, bias, eps, N.ACT_GELU_TANH, grad_mode)


# ---- GELU ------------------------------------------------------------------------------

def gelu_fwd(x):
    """y = gelu(x) (dense, x's shape) for any view x."""
    _require_cuda_f32("x", x)
    x = dense(x)
    y = torch.empty_like(x)
    N.check(N.load().oxc_gelu_fwd(x.data_ptr(), y.data_ptr(), x.numel(), _stream()), "gelu")
    return y


def gelu_bwd(x, dy):
    """dx = dy * gelu'(x), dense."""
    x, dy = dense(x), dense(dy)
    if dy.shape != x.shape:
        raise ValueError(f"shape mismatch: {list(dy.shape)} vs {list(x.shape)}")
    dx = torch.empty_like(x)
    N.check(N.load().oxc_gelu_bwd(x.data_ptr(), dy.data_ptr(), dx.data_ptr(), x.numel(),
                                  _stream()), "gelu backward")
    return dx


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x = dense(x)
        ctx.save_for_backward(x)
        return gelu_fwd(x)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        return gelu_bwd(x, dy)


def gelu(x):
    """F.gelu (functional.py:194-199): 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))),
    one fused kernel each way.  After a LayerNorm, ``layer_norm_gelu`` fuses both."""
    return _Gelu.apply(x)


# ---- softmax / log_softmax ----------------------------------------------------------

def _softmax_dim(dim, x):
    if x.dim() == 0:
        raise ValueError(f"invalid argument: dim {dim} out of range for 0-D tensor")
    d = dim + x.dim() if dim < 0 else dim
    if not 0 <= d < x.dim():
        raise ValueError(f"invalid argument: dim {dim} out of range for {x.dim()}-D tensor")
    return d


def softmax_fwd(x, log=False, dim=-1):
    """y (dense, x's shape) = softmax or log_softmax of x over `dim`; x may be
    any strided view.  Dense rows along the last dim run the row kernels,
    other layouts the strided-row or column kernels (oxc_softmax_dim_fwd)."""
    _require_cuda_f32("x", x)
    d = _softmax_dim(dim, x)
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    N.check(N.load().oxc_softmax_dim_fwd(ctypes.byref(N.make_view(x)), d, int(log), y.data_ptr(),
                                         _stream()), "softmax")
    return y


def softmax_bwd(y, dy, log=False, dim=-1):
    """dx (dense) from the forward output y (dense) and dy (any view)."""
    d = _softmax_dim(dim, y)
    dx = torch.empty(y.shape, dtype=torch.float32, device=y.device)
    N.check(N.load().oxc_softmax_dim_bwd(y.data_ptr(), ctypes.byref(N.make_view(dy)), d, int(log),
                                         dx.data_ptr(), _stream()), "softmax backward")
    return dx


class _Softmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, log, dim):
        y = softmax_fwd(x, log, dim)
        ctx.save_for_backward(y)
        ctx.log, ctx.dim = log, dim
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        return softmax_bwd(y, dy, ctx.log, ctx.dim), None, None


def softmax(x, dim=-1):
    """F.softmax (functional.py:211-215), numerically stable, over any dim."""
    return _Softmax.apply(x, False, dim)


def log_softmax(x, dim=-1):
    """F.log_softmax (functional.py:218-222) over any dim."""
    return _Softmax.apply(x, True, dim)


# ---- cross-entropy ----------------------------------------------------------------------

def _targets_tensor(targets, n, classes, device):
    """The reference takes a Python list and indexes a numpy one-hot with it
    (functional.py:285-289): the same length check and numpy's index rules."""
    if isinstance(targets, torch.Tensor):
        t = targets.to(device=device, dtype=torch.int64).reshape(-1)
        if t.numel() != n:
            raise ValueError(f"{t.numel()} targets for batch of {n}")
        return t.contiguous()
    if len(targets) != n:
        raise ValueError(f"{len(targets)} targets for batch of {n}")
    for v in targets:
        if not -classes <= int(v) < classes:
            raise IndexError(f"index {int(v)} is out of bounds for axis 1 with size {classes}")
    return torch.tensor([int(v) for v in targets], dtype=torch.int64, device=device)


def cross_entropy_fwd(logits, targets, total_rows=None):
    """Returns (loss[1], row_max, row_sum, row_nll)."""
    _require_cuda_f32("logits", logits)
    logits = _row_major("logits", logits)
    if logits.dim() != 2:
        raise ValueError(f"invalid argument: cross_entropy expects [n, classes] logits, got {list(logits.shape)}")
    n, classes = logits.shape
    t = _targets_tensor(targets, n, classes, logits.device)
    loss = torch.empty(1, dtype=torch.float32, device=logits.device)
    row_max = torch.empty(n, dtype=torch.float32, device=logits.device)
    row_sum = torch.empty_like(row_max)
    row_nll = torch.empty_like(row_max)
    flag = torch.zeros(4, dtype=torch.int32, device=logits.device)
    L = N.load()
    N.check(L.oxc_cross_entropy_fwd(logits.data_ptr(), t.data_ptr(), loss.data_ptr(),
                                    row_max.data_ptr(), row_sum.data_ptr(), row_nll.data_ptr(), n,
                                    classes, int(total_rows or n), flag.data_ptr(), _stream()),
            "cross_entropy")
    return loss, row_max, row_sum, row_nll, t, flag


def cross_entropy_bwd(logits, t, row_max, row_sum, grad_loss=None, total_rows=None):
    n, classes = logits.shape
    dlogits = torch.empty_like(logits)
    N.check(N.load().oxc_cross_entropy_bwd(
        logits.data_ptr(), t.data_ptr(), row_max.data_ptr(), row_sum.data_ptr(),
        None if grad_loss is None else grad_loss.data_ptr(), dlogits.data_ptr(), n, classes,
        int(total_rows or n), _stream()), "cross_entropy backward")
    return dlogits


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets):
        loss, row_max, row_sum, _, t, _ = cross_entropy_fwd(logits, targets)
        ctx.save_for_backward(logits, t, row_max, row_sum)
        return loss.reshape(())

    @staticmethod
    def backward(ctx, g):
        logits, t, row_max, row_sum = ctx.saved_tensors
        g = g.reshape(1).to(torch.float32).contiguous()
        return cross_entropy_bwd(logits, t, row_max, row_sum, g), None


def cross_entropy(logits, targets):
    """F.cross_entropy (functional.py:277-293): mean over the batch of
    -log_softmax(logits)[i, targets[i]]."""
    return _CrossEntropy.apply(logits, targets)


# ---- embedding ----------------------------------------------------------------------------

def _ids_tensor(indices, vocab, device):
    """The reference validates every id before copying (lib.rs:665-675):
    negative ids count from the end, anything else out of range raises."""
    if isinstance(indices, torch.Tensor):
        return indices.to(device=device, dtype=torch.int64).reshape(-1).contiguous()
    ids = [int(i) for i in indices]
    for i in ids:
        idx = vocab + i if i < 0 else i
        if idx < 0 or idx >= vocab:
            raise RuntimeError(f"out of bounds: index {i} out of range for dim 0 of size {vocab}")
    return torch.tensor(ids, dtype=torch.int64, device=device)


def embedding_fwd(ids, weight, vocab_offset=0, vocab_total=None):
    """out [n, cols] = weight[ids]; weight may be a vocab shard."""
    _require_cuda_f32("weight", weight)
    weight = _row_major("weight", weight)
    rows, cols = weight.shape
    total = int(vocab_total or rows)
    out = torch.empty(ids.numel(), cols, dtype=torch.float32, device=weight.device)
    flag = torch.zeros(4, dtype=torch.int32, device=weight.device)
    N.check(N.load().oxc_embedding_fwd(weight.data_ptr(), ids.data_ptr(), out.data_ptr(),
                                       ids.numel(), total, int(vocab_offset), rows, cols,
                                       flag.data_ptr(), _stream()), "embedding")
    return out, flag


def embedding_bwd(ids, dout, rows, vocab_offset=0, vocab_total=None):
    """dtable [rows, cols] for dout [n, cols]."""
    dout = _row_major("dout", dout)
    n, cols = ids.numel(), dout.shape[-1]
    total = int(vocab_total or rows)
    dtable = torch.empty(rows, cols, dtype=torch.float32, device=dout.device)
    flag = torch.zeros(4, dtype=torch.int32, device=dout.device)
    L = N.load()
    ws = _workspace(L.oxc_embedding_bwd_workspace_size(n, rows, cols), dout.device)
    N.check(L.oxc_embedding_bwd(dout.data_ptr(), ids.data_ptr(), dtable.data_ptr(), n, total,
                                int(vocab_offset), rows, cols, flag.data_ptr(), ws.data_ptr(),
                                ws.numel(), _stream()), "embedding backward")
    return dtable, flag


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight):
        out, _ = embedding_fwd(ids, weight)
        ctx.save_for_backward(ids)
        ctx.rows = weight.shape[0]
        return out

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        dtable, _ = embedding_bwd(ids, dense(dout), ctx.rows)
        return None, dtable


def embedding(indices, weight):
    """F.embedding (functional.py:245-247): weight.index_select(0, indices);
    indices is a flat list of ints (or an int tensor); the output is
    [len(indices), dim]."""
    _require_cuda_f32("weight", weight)
    ids = _ids_tensor(indices, weight.shape[0], weight.device)
    return _Embedding.apply(ids, weight)


# ---- SiLU / SwiGLU -----------------------------------------------------------------------

def _as2d(name, t):
    _require_cuda_f32(name, t)
    if t.dim() == 1:
        return t.reshape(1, -1)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t


def swiglu_fwd(gate, up=None, row_stats=False):
    """h = silu(gate) * up (silu(gate) if up is None) for 2-D views of any
    strides; with row_stats also the dim-1 sum, max and argmax of h."""
    g = _as2d("gate", gate)
    u = None if up is None else _as2d("up", up)
    R, C = g.shape
    h = torch.empty(R, C, dtype=torch.float32, device=g.device)
    stats = [torch.empty(R, dtype=torch.float32, device=g.device) for _ in range(3)] if row_stats else [None] * 3
    N.check(N.load().oxc_swiglu_fwd(ctypes.byref(N.make_view(g)),
                                    None if u is None else ctypes.byref(N.make_view(u)),
                                    h.data_ptr(), *[None if t is None else t.data_ptr() for t in stats],
                                    _stream()), "swiglu")
    return (h, *stats) if row_stats else h


def swiglu_bwd(gate, up, dh, sumsq=False):
    """(dgate, dup[, sum of squares of both as a 0-d f64 tensor])."""
    g = _as2d("gate", gate)
    u = None if up is None else _as2d("up", up)
    d = _as2d("dh", dh)
    R, C = g.shape
    dg = torch.empty(R, C, dtype=torch.float32, device=g.device)
    du = None if u is None else torch.empty(R, C, dtype=torch.float32, device=g.device)
    L = N.load()
    sq = torch.empty((), dtype=torch.float64, device=g.device) if sumsq else None
    ws = _workspace(L.oxc_swiglu_bwd_workspace_size(R, C) if sumsq else 0, g.device)
    N.check(L.oxc_swiglu_bwd(ctypes.byref(N.make_view(g)),
                             None if u is None else ctypes.byref(N.make_view(u)),
                             ctypes.byref(N.make_view(d)), dg.data_ptr(),
                             None if du is None else du.data_ptr(),
                             None if sq is None else sq.data_ptr(), ws.data_ptr(), ws.numel(),
                             _stream()), "swiglu backward")
    return (dg, du, sq) if sumsq else (dg, du)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        ctx.shape = gate.shape
        h = swiglu_fwd(gate, up)
        return h.reshape(gate.shape)

    @staticmethod
    def backward(ctx, dh):
        gate, up = ctx.saved_tensors
        dg, du = swiglu_bwd(gate, up, dh)
        return dg.reshape(ctx.shape), du.reshape(ctx.shape)


class _SiLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return swiglu_fwd(x).reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        dg, _ = swiglu_bwd(x, None, dy)
        return dg.reshape(x.shape)


def silu(x):
    """F.silu (functional.py:202-204): x * sigmoid(x)."""
    return _SiLU.apply(x)


def swiglu(gate, up):
    """silu(gate) * up, the decoder-MLP gate (composed by callers of F.silu)."""
    return _SwiGLU.apply(gate, up)


# ---- layers of a recurrent draft model -------------------------------------------------
#
# What a small recurrent language model needs beside the layers above when it is
# distilled from a larger one and then drafts tokens for it.  The reference has
# no counterpart.  Activations and logits may be float32 or bfloat16; the
# residual stream, weights, recurrent states, scales and probabilities are
# float32, and so is all arithmetic (a bfloat16 result is rounded once; the gradient
# of distill_loss a second time by a factor on the loss).  Their gradients cannot
# be differentiated again, and none has a forward-mode derivative: either is
# refused.

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16}


def _dtype_id(name, t):
    """The dtype id of a float32 / bfloat16 CUDA tensor on the current device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if not t.is_cuda:
        raise ValueError(f"invalid argument: {name} must live on a CUDA device "
                         "(oxitorch_b200 has no CPU path)")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"invalid argument: {name} lives on {t.device}, the current device is "
                         f"cuda:{torch.cuda.current_device()}")
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"invalid argument: {name} must be float32 or bfloat16, got {t.dtype}")
    return dt


def _operand(name, t, shape, dtype, device):
    """Checks one more tensor of a call: its shape, type and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.device != device:
        raise ValueError(f"invalid argument: {name} must live on {device}, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"invalid argument: {name} must be {str(dtype)[6:]}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"shape mismatch: {name} {list(t.shape)} vs {list(shape)}")


def _flag(t, device):
    """Checks an error flag: four dense int32."""
    _operand("flag", t, (4,), torch.int32, device)
    if not t.is_contiguous():
        raise ValueError("invalid argument: flag must be contiguous")


def _dense_any(t):
    if t.is_contiguous():
        return t
    return dense(t) if t.dtype == torch.float32 else t.contiguous()


def _rows2d(t):
    """t as [rows, cols] over its last dim with any row stride; a copy only if
    the leading dims do not collapse or the last one is not dense."""
    cols = t.shape[-1]
    if t.dim() != 2:
        try:
            t = t.view(-1, cols) if cols else t.reshape(0, 0)
        except RuntimeError:
            t = _dense_any(t).view(-1, cols)
    if cols > 1 and t.stride(1) != 1:
        t = _dense_any(t)
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _has_tangent(*tensors):
    """Whether forward-mode differentiation runs through one of them.  Then a call goes
    through its autograd function, which refuses, or refuses itself: the kernels would
    drop the tangent, and a missing one counts as zero."""
    for t in tensors:  # (0.3 us each; a generator costs another 0.5)
        if unpack_dual(t).tangent is not None:
            return True
    return False


# ---- residual addition + RMSNorm ---------------------------------------------------------

def _add_rms_args(x, residual, weight):
    dt = _dtype_id("x", x)
    if x.dim() == 0:
        raise ValueError("invalid argument: dim -1 out of range for 0-D tensor")
    _operand("residual", residual, x.shape, torch.float32, x.device)
    _operand("weight", weight, (x.shape[-1],), torch.float32, x.device)
    return dt, _rows2d(x), _rows2d(residual), dense(weight)


def add_rms_norm_fwd(x, residual, weight, eps=1e-6):
    """Returns (y, r, rstd): r = x + residual (float32), y = rms_norm(r) * weight
    in x's type, rstd the saved row factor."""
    dt, x2, res2, w = _add_rms_args(x, residual, weight)
    rows, cols = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    N.check(N.load().oxc_add_rms_norm_fwd(
        x2.data_ptr(), x2.stride(0), res2.data_ptr(), res2.stride(0), w.data_ptr(), y.data_ptr(),
        r.data_ptr(), rstd.data_ptr(), rows, cols, dt, float(eps), _stream()), "add_rms_norm")
    return y, r, rstd


def add_rms_norm_bwd(r, weight, rstd, dy, dr=None, grad_mode="ref"):
    """Returns (dx, dresidual, dweight) for dy (the type of y) and dr (float32,
    None = zero); in float32 dx and dresidual are one tensor."""
    _dtype_id("dy", dy)
    if dy.dim() == 0:
        raise ValueError("invalid argument: dim -1 out of range for 0-D tensor")
    if grad_mode not in _MODES:
        raise ValueError(f"invalid argument: unknown grad mode {grad_mode!r}")
    _operand("r", r, dy.shape, torch.float32, dy.device)
    _operand("weight", weight, (dy.shape[-1],), torch.float32, dy.device)
    _operand("rstd", rstd, dy.shape[:-1], torch.float32, dy.device)
    if dr is not None:
        _operand("dr", dr, r.shape, torch.float32, r.device)
    return _add_rms_norm_bwd(dense(r), dense(weight), dense(rstd), dy, dr, grad_mode)


def _add_rms_norm_bwd(r, w, rstd, dy, dr, grad_mode):
    dt, dy2 = _DTYPES[dy.dtype], _rows2d(dy)
    rows, cols = dy2.shape
    if dr is not None:
        dr = _rows2d(dr)
    dres = torch.empty_like(r)
    dx = dres if dt == N.F32 else torch.empty(r.shape, dtype=dy.dtype, device=r.device)
    dw = torch.empty_like(w)
    L = N.load()
    ws = _workspace(L.oxc_add_rms_norm_bwd_workspace_size(rows, cols), r.device)
    N.check(L.oxc_add_rms_norm_bwd(
        r.data_ptr(), w.data_ptr(), rstd.data_ptr(), dy2.data_ptr(), dy2.stride(0), _ptr(dr),
        0 if dr is None else dr.stride(0), dres.data_ptr(), dx.data_ptr(), dw.data_ptr(), rows,
        cols, dt, _MODES[grad_mode], ws.data_ptr(), ws.numel(), _stream()),
        "add_rms_norm backward")
    return dx, dres, dw


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, grad_mode):
        y, r, rstd = add_rms_norm_fwd(x, residual, weight, eps)
        ctx.save_for_backward(r, weight, rstd)
        ctx.grad_mode, ctx.dtype = grad_mode, x.dtype
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr):
        r, weight, rstd = ctx.saved_tensors
        if dy is None:  # only the residual stream was used
            if dr is None:
                return None, None, None, None, None
            return dr.to(ctx.dtype), dr, torch.zeros_like(weight), None, None
        return *_add_rms_norm_bwd(r, dense(weight), rstd, dy, dr, ctx.grad_mode), None, None


def add_rms_norm(x, residual, weight, eps=1e-6, grad_mode="ref"):
    """The residual's addition and the norm after it in one kernel each way:
    returns (y, r) with r = x + residual and y = rms_norm(r, weight, eps).

    x [..., cols] is float32 or bfloat16 and y has its type; residual and r, the
    residual stream, and weight [cols] are float32.  Rows may be strided."""
    if grad_mode not in _MODES:
        raise ValueError(f"invalid argument: unknown grad mode {grad_mode!r}")
    return _AddRMSNorm.apply(x, residual, weight, eps, grad_mode)


def add_rms_norm_quant(x, residual, weight, eps=1e-6, block=128):
    """add_rms_norm with y in 8 bits: returns (q, scale, r).

    Each row is cut into blocks of 128 columns (``block=None``: one block a
    row); scale [..., blocks] is max(amax(|y|) / 448, 2^-126) of a block and q,
    of type float8_e4m3fn, is y / scale rounded to nearest, so y is q * scale.
    For inference: it has no gradient, and where one is recorded an argument that
    requires it is refused (r would be cut from it)."""
    dt, x2, res2, w = _add_rms_args(x, residual, weight)
    if block not in (128, None):
        raise ValueError(f"invalid argument: block must be 128 or None, got {block}")
    if (torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad)
            or _has_tangent(x, residual, weight)):
        raise ValueError("invalid argument: add_rms_norm_quant has no gradient; train with add_rms_norm")
    rows, cols = x2.shape
    blocks = -(-cols // block) if block else 1
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(*x.shape[:-1], blocks, dtype=torch.float32, device=x.device)
    r = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    N.check(N.load().oxc_add_rms_norm_quant(
        x2.data_ptr(), x2.stride(0), res2.data_ptr(), res2.stride(0), w.data_ptr(), q.data_ptr(),
        scale.data_ptr(), r.data_ptr(), rows, cols, block or 0, dt, float(eps), _stream()),
        "add_rms_norm_quant")
    return q, scale, r


# ---- gated linear recurrence ---------------------------------------------------------------

def _sequence(t):
    """A [batch, length, dim] operand whose last dim is dense; others are copied."""
    return t if t.shape[2] <= 1 or t.stride(2) == 1 else _dense_any(t)


def _starts_tensor(starts, x):
    if starts is None:
        return None
    if isinstance(starts, torch.Tensor) and starts.dtype == torch.bool:
        starts = starts.view(torch.uint8)
    _operand("starts", starts, x.shape[:2], torch.uint8, x.device)
    return starts.contiguous()


def gated_scan_fwd(x, gate, h0=None, starts=None, save=True):
    """Returns (h, last, carry); carry (None without ``save``) is what the VJP needs."""
    dt = _dtype_id("x", x)
    if x.dim() != 3:
        raise ValueError(f"invalid argument: gated_scan expects [batch, length, dim], got {list(x.shape)}")
    _operand("gate", gate, x.shape, x.dtype, x.device)
    B, T, D = x.shape
    x, gate, starts = _sequence(x), _sequence(gate), _starts_tensor(starts, x)
    if h0 is not None:
        _operand("h0", h0, (B, D), torch.float32, x.device)
        h0 = dense(h0)
    L = N.load()
    h = torch.empty(B, T, D, dtype=x.dtype, device=x.device)
    last = torch.empty(B, D, dtype=torch.float32, device=x.device)
    carry = None
    if save:
        carry = torch.empty(L.oxc_gated_scan_carry_size(B, T, D), dtype=torch.float32, device=x.device)
    ws = _workspace(L.oxc_gated_scan_workspace_size(B, T, D), x.device)
    N.check(L.oxc_gated_scan_fwd(
        x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1),
        _ptr(starts), _ptr(h0), h.data_ptr(), last.data_ptr(), _ptr(carry), B, T, D, dt,
        ws.data_ptr(), ws.numel(), _stream()), "gated_scan")
    return h, last, carry


def gated_scan_bwd(x, gate, carry, dh=None, dlast=None, starts=None):
    """Returns (dx, dgate, dh0) for the gradients of h and of the last state
    (None = zero); carry is gated_scan_fwd's for the same shape."""
    dt = _dtype_id("x", x)
    if x.dim() != 3:
        raise ValueError(f"invalid argument: gated_scan expects [batch, length, dim], got {list(x.shape)}")
    B, T, D = x.shape
    L = N.load()
    _operand("gate", gate, x.shape, x.dtype, x.device)
    _operand("carry", carry, (L.oxc_gated_scan_carry_size(B, T, D),), torch.float32, x.device)
    if not carry.is_contiguous():
        raise ValueError("invalid argument: carry must be contiguous")
    x, gate, starts = _sequence(x), _sequence(gate), _starts_tensor(starts, x)
    if dh is not None:
        _operand("dh", dh, x.shape, x.dtype, x.device)
        dh = _sequence(dh)
    if dlast is not None:
        _operand("dlast", dlast, (B, D), torch.float32, x.device)
        dlast = dense(dlast)
    dx = torch.empty(B, T, D, dtype=x.dtype, device=x.device)
    dgate = torch.empty_like(dx)
    dh0 = torch.empty(B, D, dtype=torch.float32, device=x.device)
    ws = _workspace(L.oxc_gated_scan_workspace_size(B, T, D), x.device)
    dsb, dst = (0, 0) if dh is None else dh.stride()[:2]
    N.check(L.oxc_gated_scan_bwd(
        x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1),
        _ptr(starts), carry.data_ptr(), _ptr(dh), dsb, dst, _ptr(dlast), dx.data_ptr(),
        dgate.data_ptr(), dh0.data_ptr(), B, T, D, dt, ws.data_ptr(), ws.numel(), _stream()),
        "gated_scan backward")
    return dx, dgate, dh0


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, starts):
        h, last, carry = gated_scan_fwd(x, gate, h0, starts)
        ctx.save_for_backward(x, gate, carry, starts)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        x, gate, carry, starts = ctx.saved_tensors
        if dh is None and dlast is None:
            return None, None, None, None
        dx, dgate, dh0 = gated_scan_bwd(x, gate, carry, dh, dlast, starts)
        return dx, dgate, dh0 if ctx.needs_input_grad[2] else None, None


def gated_scan(x, gate, h0=None, starts=None):
    """The gated linear recurrence over dim 1 of x [batch, length, dim]:
    h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid(gate).  Returns (h, last),
    last [batch, dim] being the state after the last token.

    x and gate have one type (float32 or bfloat16) and any batch and time
    strides, so halves of one projection need no copy; the state h0 (zero if
    None) and last are float32.  ``starts`` (bool [batch, length]) marks where a
    new sequence begins in a packed row: the state before such a token is zero."""
    grads = (x, gate) if h0 is None else (x, gate, h0)
    if (torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in grads)
            or _has_tangent(*grads)):
        return _GatedScan.apply(x, gate, h0, starts)
    return gated_scan_fwd(x, gate, h0, starts, save=False)[:2]


def gated_step(x, gate, state, out=None):
    """One token of gated_scan for x, gate [batch, dim]: writes the state after
    it to ``out`` (``state`` itself if None) and returns h, that state in x's
    type.  For inference: it has no gradient."""
    dt = _dtype_id("x", x)
    if x.dim() != 2:
        raise ValueError(f"invalid argument: gated_step expects [batch, dim], got {list(x.shape)}")
    _operand("gate", gate, x.shape, x.dtype, x.device)
    _operand("state", state, x.shape, torch.float32, x.device)
    if out is None:
        out = state
    else:
        _operand("out", out, x.shape, torch.float32, x.device)
    if not (state.is_contiguous() and out.is_contiguous()):
        raise ValueError("invalid argument: state and out must be contiguous")
    if 0 < abs(out.data_ptr() - state.data_ptr()) < 4 * state.numel():
        raise ValueError("invalid argument: out must be state or not overlap it")
    if (torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or state.requires_grad)
            or _has_tangent(x, gate, state)):
        raise ValueError("invalid argument: gated_step has no gradient; train with gated_scan")
    x, gate = _rows2d(x), _rows2d(gate)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    N.check(N.load().oxc_gated_step(
        x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0), state.data_ptr(),
        out.data_ptr(), h.data_ptr(), x.shape[0], x.shape[1], dt, _stream()), "gated_step")
    return h


# ---- distillation ------------------------------------------------------------------------

def distill_loss_fwd(logits, teacher_logits, teacher_ids, temperature=1.0, total_rows=None,
                     grad=True, grad_loss=None, flag=None):
    """Returns (loss[1], dlogits): the gradient (times grad_loss[0] if given)
    comes from the same pass; None without ``grad``."""
    dt = _dtype_id("logits", logits)
    if logits.dim() < 2:
        raise ValueError(f"invalid argument: distill_loss expects [n, classes] logits, got {list(logits.shape)}")
    if not isinstance(teacher_ids, torch.Tensor) or teacher_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("invalid argument: teacher_ids must be an int64 or int32 tensor")
    if not isinstance(teacher_logits, torch.Tensor) or teacher_logits.dtype not in _DTYPES:
        raise ValueError("invalid argument: teacher_logits must be a float32 or bfloat16 tensor")
    if teacher_ids.shape[:-1] != logits.shape[:-1] or teacher_ids.dim() != logits.dim():
        raise ValueError(f"shape mismatch: teacher_ids {list(teacher_ids.shape)} vs logits {list(logits.shape)}")
    tl = _dense_any(teacher_logits.detach()).to(torch.float32)
    ti = teacher_ids.to(torch.int64).contiguous()
    _operand("teacher_ids", ti, ti.shape, torch.int64, logits.device)
    _operand("teacher_logits", tl, ti.shape, torch.float32, logits.device)
    if grad_loss is not None:
        one = isinstance(grad_loss, torch.Tensor) and grad_loss.numel() == 1
        _operand("grad_loss", grad_loss, grad_loss.shape if one else (1,), torch.float32, logits.device)
    if flag is not None:
        _flag(flag, logits.device)
    x = _rows2d(logits)
    rows, vocab = x.shape
    loss = torch.empty(1, dtype=torch.float32, device=x.device)
    row_loss = torch.empty(rows * N.DISTILL_PARTS, dtype=torch.float32, device=x.device)
    dlogits = torch.empty(logits.shape, dtype=x.dtype, device=x.device) if grad else None
    N.check(N.load().oxc_distill_loss(
        x.data_ptr(), x.stride(0), tl.data_ptr(), ti.data_ptr(), ti.shape[-1], float(temperature),
        _ptr(grad_loss), loss.data_ptr(), row_loss.data_ptr(), _ptr(dlogits), rows, vocab,
        int(total_rows or rows), dt, _ptr(flag), _stream()), "distill_loss")
    return loss, dlogits


class _DistillLoss(torch.autograd.Function):
    """The forward pass leaves the gradient for a loss gradient of 1; backward
    hands it out, scaled in place on the device if it is another.  A second
    backward (retain_graph) computes it again and scales it likewise, so that the
    bits do not depend on which one asks.  In bfloat16 a factor that is no power of
    two rounds the gradient a second time, by up to half a unit in its last place:
    the first rounding came before the factor was known."""

    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_ids, temperature, total_rows):
        loss, ctx.dlogits = distill_loss_fwd(logits, teacher_logits, teacher_ids, temperature, total_rows)
        ctx.save_for_backward(logits, teacher_logits, teacher_ids)
        ctx.args = temperature, total_rows
        return loss.reshape(())

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if g.dtype != torch.float32:
            g = g.to(torch.float32)
        d, ctx.dlogits = ctx.dlogits, None
        if d is None:
            d = distill_loss_fwd(*ctx.saved_tensors, *ctx.args)[1]
        N.check(N.load().oxc_scale_by(d.data_ptr(), d.numel(), _DTYPES[d.dtype], g.data_ptr(),
                                      _stream()), "distill_loss backward")
        return d, None, None, None, None


def distill_loss(logits, teacher_logits, teacher_ids, temperature=1.0, total_rows=None):
    """Distillation from a teacher's top logits: temperature^2 times the mean over
    rows of KL(p || q), p the softmax of teacher_logits / temperature over the
    row's entries and q the student's softmax of logits / temperature over the
    whole vocabulary.

    logits [..., vocab] float32 or bfloat16; teacher_logits and teacher_ids
    (int64 or int32) [..., top] with the same leading dims.  An entry with a
    negative id or a -inf logit is absent; a row without entries adds 0 to the
    mean and has a zero gradient.  An id >= vocab makes the loss NaN.
    total_rows: the divisor of the mean (the rows of this call if None), as in
    a sharded batch.  The gradient reaches logits only; in bfloat16 it is rounded
    for a factor of 1 on the loss and again when another one scales it."""
    if (torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad
            or _has_tangent(logits, teacher_logits)):
        return _DistillLoss.apply(logits, teacher_logits, teacher_ids, temperature, total_rows)
    return distill_loss_fwd(logits, teacher_logits, teacher_ids, temperature, total_rows,
                            grad=False)[0].reshape(())


# ---- verification of drafted tokens --------------------------------------------------------

def verify_draft(target, draft, tokens, uniform, race, lengths=None, flag=None):
    """Which drafted tokens the target keeps, and the token after them, from given
    random numbers.  Returns (out [batch, drafted + 1], accepted [batch]), int64.

    target [batch, drafted + 1, vocab] and draft [batch, drafted, vocab] are
    float32 probabilities (None for draft: each token was drafted with
    probability 1); tokens [batch, drafted] int64, of which lengths[b] (all if
    None) count.  Token k is kept while uniform[b, k] * q < p.  out[b] holds the
    accepted[b] kept tokens, then the token sampled after them as the first
    argmax of max(p - q, 0) / race[b] (p / race[b] when all were kept or nothing
    is left), then -1.  uniform [batch, drafted] is in [0, 1); race [batch,
    vocab] holds exponential variates (one of zero makes the quotient of a
    positive weight infinite; a token without weight is never chosen).  Tokens
    outside the vocabulary are not kept, and recorded in ``flag`` (int32[4], zeroed by the caller) if given."""
    _require_cuda_f32("target", target)
    _dtype_id("target", target)
    if target.dim() != 3 or target.shape[1] < 1:
        raise ValueError("invalid argument: verify_draft expects target [batch, drafted + 1, vocab], "
                         f"got {list(target.shape)}")
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    dev = target.device
    if draft is not None:
        _operand("draft", draft, (B, K, V), torch.float32, dev)
        draft = _sequence(draft)
    _operand("tokens", tokens, (B, K), torch.int64, dev)
    _operand("uniform", uniform, (B, K), torch.float32, dev)
    _operand("race", race, (B, V), torch.float32, dev)
    if lengths is not None:
        _operand("lengths", lengths, (B,), torch.int64, dev)
        lengths = lengths.contiguous()
    if flag is not None:
        _flag(flag, dev)
    target, tokens, uniform, race = _sequence(target), tokens.contiguous(), dense(uniform), dense(race)
    out = torch.empty(B, K + 1, dtype=torch.int64, device=dev)
    accepted = torch.empty(B, dtype=torch.int64, device=dev)
    qsb, qsk = (0, 0) if draft is None else draft.stride()[:2]
    N.check(N.load().oxc_verify_draft(
        target.data_ptr(), target.stride(0), target.stride(1), _ptr(draft), qsb, qsk,
        tokens.data_ptr(), _ptr(lengths), uniform.data_ptr(), race.data_ptr(), B, K, V,
        out.data_ptr(), accepted.data_ptr(), _ptr(flag), _stream()), "verify_draft")
    return out, accepted


# ---- layers and losses of a selective state space model ----------------------------------
#
# What a model with selective state space layers needs beside the draft model's
# operators above, in training and a token at a time; types, strides and gradients
# as there.

_ACTIVATIONS = {None: 0, "silu": 1}


def _sequences(name, x):
    dt = _dtype_id("x", x)
    if x.dim() != 3:
        raise ValueError(f"invalid argument: {name} expects [batch, length, dim], got {list(x.shape)}")
    return dt


def _recorded(*tensors):
    """Whether autograd has to see a call on these tensors."""
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    # tangents exist only within a level of forward-mode differentiation
    return forward_ad._current_level >= 0 and _has_tangent(*[t for t in tensors if isinstance(t, torch.Tensor)])


def _once(backward):
    """once_differentiable, entered only where a gradient of the gradient is recorded."""
    refusing = once_differentiable(backward)

    def run(ctx, *grads):
        return (refusing if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


def _fits(name, t, shape, dtype, device):
    """_operand, with the checks that a fitting tensor passes first: a step takes ten of them."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape
            or t.get_device() != device.index):
        _operand(name, t, shape, dtype, device)


def _lines(t):
    """A [rows, cols] operand whose last dim is dense; others are copied."""
    return t if t.stride(1) == 1 else _rows2d(t)


def _flat(t):
    """A float32 operand that is dense, None or copied."""
    return t if t is None or t.is_contiguous() else dense(t)


def _scratch(nbytes, device):
    """(tensor, address, bytes) of a workspace; nothing where none is needed."""
    if not nbytes:
        return None, None, 0
    ws = _workspace(nbytes, device)
    return ws, ws.data_ptr(), ws.numel()


def _dense_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


# ---- short causal convolution --------------------------------------------------------------

def _conv_args(name, x, shape, weight, bias, x0, activation):
    dim = shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"invalid argument: {name} expects weight [dim, width]")
    width = weight.shape[1]
    _fits("weight", weight, (dim, width), torch.float32, x.device)
    if width < 1:
        raise ValueError(f"invalid argument: {name} needs at least one tap")
    if bias is not None:
        _fits("bias", bias, (dim,), torch.float32, x.device)
    if x0 is not None:
        _fits("x0", x0, (shape[0], width - 1, dim), x.dtype, x.device)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"invalid argument: unknown activation {activation!r}")
    return width


def causal_conv_fwd(x, weight, bias=None, x0=None, starts=None, activation="silu"):
    """Returns (y, last)."""
    dt = _sequences("causal_conv", x)
    width = _conv_args("causal_conv", x, x.shape, weight, bias, x0, activation)
    B, T, D = x.shape
    x, starts = _sequence(x), _starts_tensor(starts, x)
    weight, bias = _flat(weight), _flat(bias)
    x0 = None if x0 is None else _dense_any(x0)
    y, last = _dense_like(x), x.new_empty((B, width - 1, D))
    N.check(N.load().oxc_causal_conv_fwd(
        x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _ptr(bias), _ptr(x0),
        _ptr(starts), y.data_ptr(), last.data_ptr(), B, T, D, width, _ACTIVATIONS[activation], dt,
        _stream()), "causal_conv")
    return y, last


def causal_conv_bwd(x, weight, bias=None, x0=None, dy=None, dlast=None, starts=None, activation="silu"):
    """Returns (dx, dweight, dbias, dx0) for the gradients of y and of last (None = zero)."""
    _sequences("causal_conv", x)
    width = _conv_args("causal_conv", x, x.shape, weight, bias, x0, activation)
    if dy is not None:
        _fits("dy", dy, x.shape, x.dtype, x.device)
    if dlast is not None:
        _fits("dlast", dlast, (x.shape[0], width - 1, x.shape[2]), x.dtype, x.device)
    return _causal_conv_bwd(x, weight, bias, x0, dy, dlast, _starts_tensor(starts, x), activation)


def _causal_conv_bwd(x, weight, bias, x0, dy, dlast, starts, activation):
    (B, T, D), width, dev = x.shape, weight.shape[1], x.device
    x, weight, bias = _sequence(x), _flat(weight), _flat(bias)
    x0 = None if x0 is None else _dense_any(x0)
    dy = None if dy is None else _sequence(dy)
    dlast = None if dlast is None else _dense_any(dlast)
    dx, dx0, dw = _dense_like(x), x.new_empty((B, width - 1, D)), weight.new_empty(D * (width + 1))
    L = N.load()
    ws = _workspace(L.oxc_causal_conv_bwd_workspace_size(B, T, D, width), dev)
    ysb, yst = (0, 0) if dy is None else dy.stride()[:2]
    xsb, xst, _ = x.stride()
    N.check(L.oxc_causal_conv_bwd(
        x.data_ptr(), xsb, xst, weight.data_ptr(), _ptr(bias), _ptr(x0), _ptr(starts), _ptr(dy), ysb,
        yst, _ptr(dlast), dx.data_ptr(), dx0.data_ptr(), dw.data_ptr(), B, T, D, width,
        _ACTIVATIONS[activation], _DTYPES[x.dtype], ws.data_ptr(), ws.numel(), _stream()),
        "causal_conv backward")
    dw, db = dw.split((D * width, D))
    return dx, dw.view(D, width), db, dx0


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, x0, starts, activation):
        y, last = causal_conv_fwd(x, weight, bias, x0, starts, activation)
        starts = _starts_tensor(starts, x)
        ctx.save_for_backward(x, weight, bias, x0, starts)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @_once
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return None, None, None, None, None, None
        x, weight, bias, x0, starts = ctx.saved_tensors
        dx, dw, db, dx0 = _causal_conv_bwd(x, weight, bias, x0, dy, dlast, starts, ctx.activation)
        return dx, dw, None if bias is None else db, None if x0 is None else dx0, None, None


def causal_conv(x, weight, bias=None, x0=None, starts=None, activation="silu"):
    """A short causal convolution over dim 1 of x [batch, length, dim], channel by
    channel: u_t = bias + sum_k weight[:, k] x_{t - width + 1 + k}, y = silu(u)
    (``activation=None``: u).  Returns (y, last).

    x is float32 or bfloat16 with any batch and time strides; weight [dim, width],
    width 1 to 8, and bias [dim] are float32.  x0 [batch, width - 1, dim], of x's
    type, holds the inputs before the first token (zeros if None), and last the
    ones that a continuation of the rows takes as its x0.  ``starts`` (bool [batch,
    length]) marks where a new sequence begins in a packed row: taps do not reach
    before it, and last is zero there."""
    if _recorded(x, weight, bias, x0):
        return _CausalConv.apply(x, weight, bias, x0, starts, activation)
    return causal_conv_fwd(x, weight, bias, x0, starts, activation)


def causal_conv_step(x, weight, bias, state, out=None, activation="silu"):
    """One token of causal_conv for x [batch, dim] after the inputs in state [batch,
    width - 1, dim]: returns y and writes the inputs for the next token to ``out``
    (``state`` itself if None).  For inference: it has no gradient."""
    dt = _dtype_id("x", x)
    if x.dim() != 2:
        raise ValueError(f"invalid argument: causal_conv_step expects [batch, dim], got {list(x.shape)}")
    width = _conv_args("causal_conv_step", x, x.shape, weight, bias, None, activation)
    _fits("state", state, (x.shape[0], width - 1, x.shape[1]), x.dtype, x.device)
    out = _state_out(state, out)
    if _recorded(x, weight, bias, state):
        raise ValueError("invalid argument: causal_conv_step has no gradient; train with causal_conv")
    x, weight, bias = _lines(x), _flat(weight), _flat(bias)
    y = _dense_like(x)
    N.check(N.load().oxc_causal_conv_step(
        x.data_ptr(), x.stride(0), weight.data_ptr(), _ptr(bias), state.data_ptr(), out.data_ptr(),
        y.data_ptr(), x.shape[0], x.shape[1], width, _ACTIVATIONS[activation], dt, _stream()),
        "causal_conv_step")
    return y


def _state_out(state, out):
    """Where a step writes the state after it: `state`, or a tensor that does not overlap it."""
    if out is None or out is state:
        out = state
    else:
        _fits("out", out, state.shape, state.dtype, state.device)
    if not (state.is_contiguous() and out.is_contiguous()):
        raise ValueError("invalid argument: state and out must be contiguous")
    if 0 < abs(out.data_ptr() - state.data_ptr()) < state.element_size() * state.numel():
        raise ValueError("invalid argument: out must be state or not overlap it")
    return out


# ---- selective state space scan ------------------------------------------------------------

def _selective_args(x, lead, delta, A, B, C, D, z, delta_bias):
    """Checks everything but x and the states; `lead`: x's dims before the last."""
    dim, dev = x.shape[-1], x.device
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise ValueError("invalid argument: A must be [dim, state]")
    n = A.shape[1]
    _fits("delta", delta, x.shape, x.dtype, dev)
    _fits("A", A, (dim, n), torch.float32, dev)
    _fits("B", B, (*lead, n), x.dtype, dev)
    _fits("C", C, (*lead, n), x.dtype, dev)
    if D is not None:
        _fits("D", D, (dim,), torch.float32, dev)
    if z is not None:
        _fits("z", z, x.shape, x.dtype, dev)
    if delta_bias is not None:
        _fits("delta_bias", delta_bias, (dim,), torch.float32, dev)
    return n


def selective_scan_fwd(x, delta, A, B, C, D=None, z=None, delta_bias=None, h0=None, starts=None,
                       save=True):
    """Returns (y, last, carry); carry (None without ``save``) is what the VJP needs."""
    dt = _sequences("selective_scan", x)
    batch, length, dim = x.shape
    n = _selective_args(x, (batch, length), delta, A, B, C, D, z, delta_bias)
    if h0 is not None:
        _fits("h0", h0, (batch, dim, n), torch.float32, x.device)
    x, delta, B, C, starts = _sequence(x), _sequence(delta), _sequence(B), _sequence(C), _starts_tensor(starts, x)
    z = None if z is None else _sequence(z)
    A, D, delta_bias, h0 = _flat(A), _flat(D), _flat(delta_bias), _flat(h0)
    L = N.load()
    y, last = _dense_like(x), A.new_empty((batch, dim, n))
    carry = A.new_empty(L.oxc_selective_scan_carry_size(batch, length, dim, n)) if save else None
    ws, at, nbytes = _scratch(L.oxc_selective_scan_workspace_size(batch, length, dim, n, 0), x.device)
    zsb, zst = (0, 0) if z is None else z.stride()[:2]
    N.check(L.oxc_selective_scan_fwd(
        x.data_ptr(), x.stride(0), x.stride(1), delta.data_ptr(), delta.stride(0), delta.stride(1),
        A.data_ptr(), B.data_ptr(), B.stride(0), B.stride(1), C.data_ptr(), C.stride(0), C.stride(1),
        _ptr(D), _ptr(z), zsb, zst, _ptr(delta_bias), _ptr(starts), _ptr(h0), y.data_ptr(),
        last.data_ptr(), _ptr(carry), batch, length, dim, n, dt, at, nbytes, _stream()), "selective_scan")
    return y, last, carry


def selective_scan_bwd(x, delta, A, B, C, carry, D=None, z=None, delta_bias=None, starts=None,
                       dy=None, dlast=None):
    """Returns (dx, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dh0) for the gradients of y
    and of the last state (None = zero); carry is selective_scan_fwd's.  dz is None
    without z."""
    _sequences("selective_scan", x)
    batch, length, dim = x.shape
    n = _selective_args(x, (batch, length), delta, A, B, C, D, z, delta_bias)
    _fits("carry", carry, (N.load().oxc_selective_scan_carry_size(batch, length, dim, n),), torch.float32, x.device)
    if not carry.is_contiguous():
        raise ValueError("invalid argument: carry must be contiguous")
    if dy is not None:
        _fits("dy", dy, x.shape, x.dtype, x.device)
    if dlast is not None:
        _fits("dlast", dlast, (batch, dim, n), torch.float32, x.device)
    return _selective_scan_bwd(x, delta, A, B, C, carry, D, z, delta_bias, _starts_tensor(starts, x), dy, dlast)


def _selective_scan_bwd(x, delta, A, B, C, carry, D, z, delta_bias, starts, dy, dlast):
    (batch, length, dim), n, dev = x.shape, A.shape[1], x.device
    x, delta, B, C = _sequence(x), _sequence(delta), _sequence(B), _sequence(C)
    z = None if z is None else _sequence(z)
    dy = None if dy is None else _sequence(dy)
    A, D, delta_bias, dlast = _flat(A), _flat(D), _flat(delta_bias), _flat(dlast)
    dx, ddelta, dz = _dense_like(x), _dense_like(x), None if z is None else _dense_like(x)
    dB, dC = _dense_like(B), _dense_like(B)
    sums, dh0 = A.new_empty(dim * (n + 2)), A.new_empty((batch, dim, n))
    L = N.load()
    ws = _workspace(L.oxc_selective_scan_workspace_size(batch, length, dim, n, 1), dev)
    zsb, zst = (0, 0) if z is None else z.stride()[:2]
    ysb, yst = (0, 0) if dy is None else dy.stride()[:2]
    N.check(L.oxc_selective_scan_bwd(
        x.data_ptr(), x.stride(0), x.stride(1), delta.data_ptr(), delta.stride(0), delta.stride(1),
        A.data_ptr(), B.data_ptr(), B.stride(0), B.stride(1), C.data_ptr(), C.stride(0), C.stride(1),
        _ptr(D), _ptr(z), zsb, zst, _ptr(delta_bias), _ptr(starts), carry.data_ptr(), _ptr(dy), ysb,
        yst, _ptr(dlast), dx.data_ptr(), ddelta.data_ptr(), sums.data_ptr(), dB.data_ptr(),
        dC.data_ptr(), _ptr(dz), dh0.data_ptr(), batch, length, dim, n, _DTYPES[x.dtype],
        ws.data_ptr(), ws.numel(), _stream()), "selective_scan backward")
    dA, dD, dbias = sums.split((dim * n, dim, dim))
    return dx, ddelta, dA.view(dim, n), dB, dC, dD, dz, dbias, dh0


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, h0, starts):
        y, last, carry = selective_scan_fwd(x, delta, A, B, C, D, z, delta_bias, h0, starts)
        ctx.save_for_backward(x, delta, A, B, C, carry, D, z, delta_bias, _starts_tensor(starts, x))
        ctx.has_h0 = h0 is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @_once
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return (None,) * 10
        x, delta, A, B, C, carry, D, z, delta_bias, starts = ctx.saved_tensors
        dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0 = _selective_scan_bwd(
            x, delta, A, B, C, carry, D, z, delta_bias, starts, dy, dlast)
        return (dx, ddelta, dA, dB, dC, None if D is None else dD, dz,
                None if delta_bias is None else dbias, dh0 if ctx.has_h0 else None, None)


def selective_scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, h0=None, starts=None):
    """The selective state space scan over dim 1 of x [batch, length, dim]: with dt =
    softplus(delta + delta_bias), the state h [dim, state] of a sequence is
    h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t, and y_t = (sum over the states of C_t h_t
    + D x_t) silu(z_t).  Returns (y, last), last [batch, dim, state] being the state
    after the last token.

    x, delta and z [batch, length, dim] and B and C [batch, length, state] have one type
    (float32 or bfloat16) and any batch and time strides, so parts of one projection
    need no copy; A [dim, state] (negative for a state that decays; state up to 128), D and
    delta_bias [dim], the state h0 (zero if None) and last are float32.  D, z and
    delta_bias may be None (no D x, no gate, no bias).  ``starts`` (bool [batch,
    length]) marks where a new sequence begins in a packed row: the state before such
    a token is zero."""
    if _recorded(x, delta, A, B, C, D, z, delta_bias, h0):
        return _SelectiveScan.apply(x, delta, A, B, C, D, z, delta_bias, h0, starts)
    return selective_scan_fwd(x, delta, A, B, C, D, z, delta_bias, h0, starts, save=False)[:2]


def selective_step(x, delta, A, B, C, state, D=None, z=None, delta_bias=None, out=None):
    """One token of selective_scan for x, delta, z [batch, dim] and B, C [batch, state]:
    writes the state after it to ``out`` (``state`` itself if None) and returns y.  For
    inference: it has no gradient."""
    dt = _dtype_id("x", x)
    if x.dim() != 2:
        raise ValueError(f"invalid argument: selective_step expects [batch, dim], got {list(x.shape)}")
    batch, dim = x.shape
    n = _selective_args(x, (batch,), delta, A, B, C, D, z, delta_bias)
    _fits("state", state, (batch, dim, n), torch.float32, x.device)
    out = _state_out(state, out)
    if _recorded(x, delta, A, B, C, state, D, z, delta_bias):
        raise ValueError("invalid argument: selective_step has no gradient; train with selective_scan")
    x, delta, B, C = _lines(x), _lines(delta), _lines(B), _lines(C)
    z = None if z is None else _lines(z)
    A, D, delta_bias = _flat(A), _flat(D), _flat(delta_bias)
    y = _dense_like(x)
    N.check(N.load().oxc_selective_step(
        x.data_ptr(), x.stride(0), delta.data_ptr(), delta.stride(0), A.data_ptr(), B.data_ptr(),
        B.stride(0), C.data_ptr(), C.stride(0), _ptr(D), _ptr(z), 0 if z is None else z.stride(0),
        _ptr(delta_bias), state.data_ptr(), out.data_ptr(), y.data_ptr(), batch, dim, n, dt,
        _stream()), "selective_step")
    return y


# ---- clipped policy loss -------------------------------------------------------------------

def _sampled_tokens(name, logits, tokens):
    dt = _dtype_id("logits", logits)
    if logits.dim() < 2:
        raise ValueError(f"invalid argument: {name} expects [n, classes] logits, got {list(logits.shape)}")
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError("invalid argument: tokens must be an int64 or int32 tensor")
    tokens = tokens.to(torch.int64).contiguous()
    _fits("tokens", tokens, logits.shape[:-1], torch.int64, logits.device)
    return dt, tokens


def _mean_divisor(name, total_rows, tokens):
    """The divisor of a mean over rows, of which those with a negative token do not count.
    One below the number of rows is compared with the rows that count, for which the host
    waits for the device; while a graph is captured their tokens are not there yet, and it
    is taken as it is."""
    rows = tokens.numel()
    if total_rows is None:
        return max(rows, 1)
    total = int(total_rows)
    if 0 < total < rows and not torch.cuda.is_current_stream_capturing():
        count = int((tokens >= 0).sum())
        if total < count:
            raise ValueError(f"invalid argument: {name}: total_rows {total} must cover the {count} rows that count")
    return total


def policy_loss_fwd(logits, tokens, old_logp, advantages, ref_logp=None, clip=0.2, kl_coef=0.0,
                    temperature=1.0, total_rows=None, grad=True, grad_loss=None, flag=None):
    """Returns (loss[1], logp, dlogits): the gradient (times grad_loss[0] if given)
    comes from the same pass; None without ``grad``."""
    dt, tok = _sampled_tokens("policy_loss", logits, tokens)
    dev, lead = logits.device, logits.shape[:-1]
    _fits("old_logp", old_logp, lead, torch.float32, dev)
    _fits("advantages", advantages, lead, torch.float32, dev)
    below, above = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (below >= 0 and above >= 0 and 0 <= kl_coef < float("inf")):
        raise ValueError(f"invalid argument: clip {clip} and kl_coef {kl_coef} must not be negative")
    if ref_logp is not None:
        _fits("ref_logp", ref_logp, lead, torch.float32, dev)
    elif kl_coef > 0:
        raise ValueError("invalid argument: the KL term needs ref_logp")
    if grad_loss is not None:
        one = isinstance(grad_loss, torch.Tensor) and grad_loss.numel() == 1
        _fits("grad_loss", grad_loss, grad_loss.shape if one else (1,), torch.float32, dev)
    if flag is not None:
        _flag(flag, dev)
    x, old, adv, ref = _rows2d(logits), dense(old_logp), dense(advantages), _flat(ref_logp)
    rows, vocab = tok.numel(), logits.shape[-1]
    total = _mean_divisor("policy_loss", total_rows, tok)
    loss, logp, row_loss = old.new_empty(1), _dense_like(old), old.new_empty(rows)
    dlogits = _dense_like(logits) if grad else None
    N.check(N.load().oxc_policy_loss(
        x.data_ptr(), x.stride(0), tok.data_ptr(), old.data_ptr(), adv.data_ptr(), _ptr(ref),
        float(below), float(above), float(kl_coef), float(temperature), _ptr(grad_loss),
        loss.data_ptr(), logp.data_ptr(), row_loss.data_ptr(), _ptr(dlogits), rows, vocab, total, dt,
        _ptr(flag), _stream()), "policy_loss")
    return loss, logp, dlogits


class _PolicyLoss(torch.autograd.Function):
    """As _DistillLoss: the forward pass leaves the gradient for a loss gradient of 1,
    backward hands it out, scaled on the device if it is another (in bfloat16 rounded a
    second time then), and a second backward computes it again."""

    @staticmethod
    def forward(ctx, logits, tokens, old_logp, advantages, ref_logp, *args):
        loss, logp, ctx.dlogits = policy_loss_fwd(logits, tokens, old_logp, advantages, ref_logp, *args)
        ctx.save_for_backward(logits, tokens, old_logp, advantages, ref_logp)
        ctx.args = args
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss.reshape(()), logp

    @staticmethod
    @_once
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 9
        if g.dtype != torch.float32:
            g = g.to(torch.float32)
        d, ctx.dlogits = ctx.dlogits, None
        if d is None:
            d = policy_loss_fwd(*ctx.saved_tensors, *ctx.args)[2]
        N.check(N.load().oxc_scale_by(d.data_ptr(), d.numel(), _DTYPES[d.dtype], g.data_ptr(),
                                      _stream()), "policy_loss backward")
        return d, None, None, None, None, None, None, None, None


def policy_loss(logits, tokens, old_logp, advantages, ref_logp=None, clip=0.2, kl_coef=0.0,
                temperature=1.0, total_rows=None):
    """The clipped policy loss of sampled tokens with a KL term towards a reference:
    returns (loss, logp), logp [...] being each token's log-probability in
    softmax(logits / temperature) (no gradient runs through it).  With r = exp(logp -
    old_logp) the loss is the mean over rows of

        -min(r A, clamp(r, 1 - clip, 1 + clip) A)
        + kl_coef (exp(ref_logp - logp) - (ref_logp - logp) - 1).

    logits [..., vocab] float32 or bfloat16; tokens [...] int64 or int32; old_logp,
    advantages A and ref_logp [...] float32, which the gradient does not reach.  clip:
    one number, or (below, above).  A row with a negative token (padding) adds 0 to the
    mean and has a zero gradient and logp; a token >= vocab makes the loss NaN.
    total_rows: the divisor of the mean (the rows of this call if None), as in a sharded
    batch, or, where only unpadded tokens count, their number: one below the rows of the
    call has to cover those that are no padding, and the host waits for the tokens to see
    that it does (not while a graph is captured).  In bfloat16 the gradient is rounded for
    a factor of 1 on the loss and again when another one scales it."""
    if _recorded(old_logp, advantages, ref_logp):
        for name, t in (("old_logp", old_logp), ("advantages", advantages), ("ref_logp", ref_logp)):
            if _recorded(t):
                raise ValueError(f"invalid argument: {name} gets no gradient; detach it")
    if _recorded(logits):
        return _PolicyLoss.apply(logits, tokens, old_logp, advantages, ref_logp, clip, kl_coef,
                                 temperature, total_rows)
    loss, logp, _ = policy_loss_fwd(logits, tokens, old_logp, advantages, ref_logp, clip, kl_coef,
                                    temperature, total_rows, grad=False)
    return loss.reshape(()), logp


def token_logprobs(logits, tokens, temperature=1.0, flag=None):
    """Each token's log-probability [...] in softmax(logits / temperature), as
    policy_loss returns it: its old_logp and ref_logp, from the logits of the policy
    that sampled the tokens and of the reference.  It has no gradient."""
    dt, tok = _sampled_tokens("token_logprobs", logits, tokens)
    if _recorded(logits):
        raise ValueError("invalid argument: token_logprobs has no gradient; train with policy_loss")
    if flag is not None:
        _flag(flag, logits.device)
    x = _rows2d(logits)
    logp = torch.empty(logits.shape[:-1], dtype=torch.float32, device=x.device)
    rows, vocab = tok.numel(), logits.shape[-1]
    N.check(N.load().oxc_policy_loss(
        x.data_ptr(), x.stride(0), tok.data_ptr(), None, None, None, 0.0, 0.0, 0.0,
        float(temperature), None, None, logp.data_ptr(), None, None, rows, vocab, max(rows, 1), dt,
        _ptr(flag), _stream()), "token_logprobs")
    return logp
