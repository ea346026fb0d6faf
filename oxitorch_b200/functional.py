"""Device-side mirror of oxitorch's ``F.*`` layer functions.

Same names, argument meaning and error behaviour as
``python/oxitorch/nn/functional.py`` for the memory-bound layers; each call is
one fused CUDA kernel through liboxicuda.so, and its VJP is one fused kernel
(plus a deterministic column-sum finisher for weight gradients).  Tensors are
torch CUDA float32 tensors: torch supplies device memory, the stream and the
autograd graph bookkeeping (``torch.autograd.Function``); all arithmetic on
the path is ours.

The last part of the file, the layers of a recurrent draft model, has no
counterpart in the reference and takes bfloat16 activations too.

``grad_mode`` selects the backward semantics of the norms:
``"ref"`` (default) reproduces the reference graph, where ``rsqrt`` is
detached (crates/oxi-bindings/src/lib.rs:682-697); ``"exact"`` is the full
mathematical gradient.
"""

from __future__ import annotations

import torch
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
