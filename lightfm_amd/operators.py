"""Operators of a full-softmax training step on tensors that live on the GPU (include/lfm_ops.h).

`LightFM` trains with sampled ranking losses from host arrays; a model that is trained with the softmax over the whole
catalogue -- a session or sequence recommender on top of the same item tables -- needs three operators more, and needs
them on device memory, between the layers of its own program.  They take and return torch tensors of one GPU:

    softmax_loss(hidden, table, targets, bias=, weights=)       -> loss, lse
    softmax_loss_grad(hidden, table, targets, bias=, weights=)  -> loss, lse, d_hidden, d_table, d_bias
    embedding_lookup(table, ids, indptr=, values=, scale=)      -> out
    embedding_lookup_grad(d_out, ids, n_rows, indptr=, values=, scale=) -> d_table
    global_norm(tensors)                                        -> norm
    clip_global_norm(tensors, max_norm, out=)                   -> norm

float32, bfloat16 and float16 tensors; ids are int32 or int64, and an id outside the table (-1 is the padding id) has no
loss, gives a zero row and gets no gradient.  Rows may be strided (`t[:, :64]`), the elements of a row are contiguous.
Everything is enqueued on torch's current stream and nothing is waited for: the calls can be captured into HIP graphs.
Results and scratch memory come from torch's allocator.  The functions compute on the values alone: they do not record
autograd history (a training loop calls the gradient functions, or wraps them in its own `autograd.Function`).

Wrong arguments raise ValueError / TypeError like the rest of the package.  There is no CPU fallback.
"""
import ctypes as C
import os

import torch

from . import _native as N

__all__ = ["softmax_loss", "softmax_loss_grad", "embedding_lookup", "embedding_lookup_grad", "global_norm",
           "clip_global_norm"]

LIB_PATH = os.path.join(os.path.dirname(N.LIB_PATH), "liblfm_ops.so")

# every symbol include/lfm_ops.h declares (tests check the .so exports them all)
EXPORTS = ("lfm_ops_last_error", "lfm_ops_softmax_workspace", "lfm_ops_softmax_loss", "lfm_ops_softmax_loss_grad",
           "lfm_ops_embedding_lookup", "lfm_ops_embedding_grad_workspace", "lfm_ops_embedding_lookup_grad",
           "lfm_ops_clip_workspace", "lfm_ops_clip_global_norm")

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}


class LfmSoftmaxArgs(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("hidden", "table", "targets", "bias", "weights", "loss", "lse", "d_hidden",
                                           "d_table", "d_bias")]
                + [(n, C.c_int64) for n in ("rows", "vocab", "hidden_stride", "table_stride")]
                + [(n, C.c_int32) for n in ("d", "dtype", "id_bytes", "reserved")])


class LfmLookupArgs(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("table", "ids", "indptr", "values", "out", "d_out")]
                + [(n, C.c_int64) for n in ("rows", "vocab", "nnz", "table_stride", "d_out_stride")]
                + [(n, C.c_int32) for n in ("d", "dtype", "id_bytes")] + [("scale", C.c_float)])


_lib = None


def lib():
    """Loads liblfm_ops.so against the HIP runtime torch uses; raises HipBackendError if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise N.HipBackendError("%s not found: build it with `python -m lightfm_amd.build` "
                                    "(the HIP backend has no CPU fallback)" % LIB_PATH)
        l = C.CDLL(LIB_PATH)
        for name in EXPORTS:
            getattr(l, name).restype = C.c_int
        l.lfm_ops_last_error.restype = C.c_char_p
        _lib = l
    return _lib


def _check(rc):
    if rc >= 0:
        return
    msg = lib().lfm_ops_last_error().decode("utf-8", "replace")
    raise {-1: ValueError, -3: MemoryError, -5: NotImplementedError}.get(rc, N.HipBackendError)(msg)


def _tensor(t, name, ndim, dtypes, device=None, dense=True):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype not in dtypes:
        raise ValueError("%s has dtype %s, expected %s" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    if t.dim() != ndim:
        raise ValueError("%s has %d dimensions, expected %d" % (name, t.dim(), ndim))
    if t.device.type != "cuda":
        raise ValueError("%s is on %s: the operators need a GPU tensor (there is no CPU fallback)" % (name, t.device))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    if dense and not t.is_contiguous():
        raise ValueError("%s is not contiguous" % name)
    return t


def _matrix(t, name, device=None, dtypes=tuple(_DTYPES)):
    """A matrix of contiguous rows; returns its row stride."""
    _tensor(t, name, 2, dtypes, device, dense=False)
    rows, d = t.shape
    if d < 1:
        raise ValueError("%s has no columns" % name)
    if d > 1 and t.stride(1) != 1 and t.numel():
        raise ValueError("the elements of a row of %s are not contiguous" % name)
    stride = t.stride(0) if rows > 1 else d
    if stride < d:
        raise ValueError("the rows of %s overlap" % name)
    return stride


class _On(object):
    """The device of a call made current (when it is not), its current stream and scratch memory."""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.guard = None
        if torch.cuda.current_device() != self.device.index:
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        self.stream = torch.cuda.current_stream(self.device).cuda_stream
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def scratch(self, nbytes):
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)


def _softmax(hidden, table, targets, bias, weights, grad):
    hs = _matrix(hidden, "hidden")
    ts = _matrix(table, "table", hidden.device, (hidden.dtype,))
    rows, d = hidden.shape
    vocab = table.shape[0]
    if table.shape[1] != d:
        raise ValueError("hidden has %d columns, table %d" % (d, table.shape[1]))
    if vocab < 1:
        raise ValueError("table has no rows")
    _tensor(targets, "targets", 1, tuple(_ID_BYTES), hidden.device)
    if targets.shape[0] != rows:
        raise ValueError("hidden has %d rows, targets %d" % (rows, targets.shape[0]))
    for extra, name, n in ((bias, "bias", vocab), (weights, "weights", rows)):
        if extra is not None:
            _tensor(extra, name, 1, (torch.float32,), hidden.device)
            if extra.shape[0] != n:
                raise ValueError("%s has %d entries, expected %d" % (name, extra.shape[0], n))
    l = lib()
    with _On(hidden.device) as on:
        loss = torch.empty(rows, dtype=torch.float32, device=hidden.device)
        lse = torch.empty_like(loss)
        a = LfmSoftmaxArgs(hidden.data_ptr(), table.data_ptr(), targets.data_ptr(),
                           None if bias is None else bias.data_ptr(), None if weights is None else weights.data_ptr(),
                           loss.data_ptr(), lse.data_ptr(), None, None, None, rows, vocab, hs, ts, d,
                           _DTYPES[hidden.dtype], _ID_BYTES[targets.dtype], 0)
        out = (loss, lse)
        if grad:
            d_hidden = torch.empty((rows, d), dtype=hidden.dtype, device=hidden.device)
            d_table = torch.empty((vocab, d), dtype=hidden.dtype, device=hidden.device)
            d_bias = None if bias is None else torch.empty(vocab, dtype=torch.float32, device=hidden.device)
            a.d_hidden, a.d_table = d_hidden.data_ptr(), d_table.data_ptr()
            a.d_bias = None if bias is None else d_bias.data_ptr()
            out = (loss, lse, d_hidden, d_table, d_bias)
        need = C.c_int64()
        _check(l.lfm_ops_softmax_workspace(C.c_int64(rows), C.c_int64(vocab), d, a.dtype, int(grad), C.byref(need)))
        ws = on.scratch(need.value)
        call = l.lfm_ops_softmax_loss_grad if grad else l.lfm_ops_softmax_loss
        _check(call(C.byref(a), C.c_void_p(ws.data_ptr()), need, C.c_void_p(on.stream)))
    return out


def softmax_loss(hidden, table, targets, bias=None, weights=None):
    """Cross entropy of every row of `hidden` [rows, d] against all rows of `table` [vocab, d]: scores
    s = hidden table^T + bias, lse = log sum exp s, loss = weights * (lse - s[target]).  Returns (loss, lse), float32
    [rows]; a row whose target is not in [0, vocab) has loss 0.  bias [vocab] / weights [rows] are float32; a bias of
    -inf takes an item out of the softmax.  The scores are never kept."""
    return _softmax(hidden, table, targets, bias, weights, False)


def softmax_loss_grad(hidden, table, targets, bias=None, weights=None):
    """softmax_loss with the gradients of the SUM of the losses: (loss, lse, d_hidden, d_table, d_bias); d_bias is None
    without a bias.  For the mean, hand in weights of 1 / rows.  Gradients have the type of hidden / table."""
    return _softmax(hidden, table, targets, bias, weights, True)


def _lookup_args(ids, indptr, values, scale, rows, vocab, d, dtype, device):
    _tensor(ids, "ids", 1, tuple(_ID_BYTES), device)
    if indptr is not None:
        _tensor(indptr, "indptr", 1, (ids.dtype,), device)
        if indptr.shape[0] < 1:
            raise ValueError("indptr is empty")
        if indptr.shape[0] == 1 and ids.shape[0]:
            raise ValueError("ids without a bag")
    if values is not None:
        if indptr is None:
            raise ValueError("values need an indptr")
        _tensor(values, "values", 1, (torch.float32,), device)
        if values.shape[0] != ids.shape[0]:
            raise ValueError("ids has %d entries, values %d" % (ids.shape[0], values.shape[0]))
    return LfmLookupArgs(None, ids.data_ptr(), None if indptr is None else indptr.data_ptr(),
                         None if values is None else values.data_ptr(), None, None, rows, vocab, ids.shape[0], d, d, d,
                         _DTYPES[dtype], _ID_BYTES[ids.dtype], float(scale))


def embedding_lookup(table, ids, indptr=None, values=None, scale=1.0):
    """Rows of `table` [vocab, d] times `scale`: out[r] = scale * table[ids[r]], or, with `indptr` [rows + 1] (CSR bags, as
    in a LightFM feature matrix), out[r] = scale * sum_j values[j] * table[ids[j]] over bag r.  values default to 1.
    Sums are float32 in the order of the bag; out has the type of table."""
    ts = _matrix(table, "table")
    vocab, d = table.shape
    if vocab < 1:
        raise ValueError("table has no rows")
    _tensor(ids, "ids", 1, tuple(_ID_BYTES), table.device)
    rows = ids.shape[0] if indptr is None else max(0, indptr.shape[0] - 1)
    a = _lookup_args(ids, indptr, values, scale, rows, vocab, d, table.dtype, table.device)
    l = lib()
    with _On(table.device) as on:
        out = torch.empty((rows, d), dtype=table.dtype, device=table.device)
        a.table, a.table_stride, a.out = table.data_ptr(), ts, out.data_ptr()
        _check(l.lfm_ops_embedding_lookup(C.byref(a), C.c_void_p(on.stream)))
    return out


def embedding_lookup_grad(d_out, ids, n_rows, indptr=None, values=None, scale=1.0):
    """Gradient of embedding_lookup with respect to its table of `n_rows` rows: d_table[v] = scale * sum of values[j] *
    d_out[r] over the places where ids[j] == v.  The ids are sorted and each row is summed in float32 in the order of
    their positions (no atomics: the same bits every time).  d_table is dense, of the type of d_out."""
    ds = _matrix(d_out, "d_out")
    rows, d = d_out.shape
    n_rows = int(n_rows)
    if n_rows < 1:
        raise ValueError("n_rows must be positive")
    a = _lookup_args(ids, indptr, values, scale, rows, n_rows, d, d_out.dtype, d_out.device)
    if rows != (ids.shape[0] if indptr is None else indptr.shape[0] - 1):
        raise ValueError("d_out has %d rows, expected %d"
                         % (rows, ids.shape[0] if indptr is None else indptr.shape[0] - 1))
    l = lib()
    with _On(d_out.device) as on:
        out = torch.empty((n_rows, d), dtype=d_out.dtype, device=d_out.device)
        a.d_out, a.d_out_stride, a.out = d_out.data_ptr(), ds, out.data_ptr()
        need = C.c_int64()
        _check(l.lfm_ops_embedding_grad_workspace(C.c_int64(rows), C.c_int64(n_rows), C.c_int64(a.nnz), d,
                                                  int(indptr is not None), C.byref(need)))
        ws = on.scratch(need.value)
        _check(l.lfm_ops_embedding_lookup_grad(C.byref(a), C.c_void_p(ws.data_ptr()), need, C.c_void_p(on.stream)))
    return out


def _clip(tensors, max_norm, out, scale):
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors")
    device = tensors[0].device if isinstance(tensors[0], torch.Tensor) else None
    for i, t in enumerate(tensors):
        _tensor(t, "tensors[%d]" % i, t.dim() if isinstance(t, torch.Tensor) else 0, tuple(_DTYPES), device)
    n = len(tensors)
    outs = None
    if scale:
        outs = tensors
        if out is not None:
            outs = list(out)
            if len(outs) != n:
                raise ValueError("%d tensors, %d outputs" % (n, len(outs)))
            for i, (t, o) in enumerate(zip(tensors, outs)):
                _tensor(o, "out[%d]" % i, t.dim(), (t.dtype,), device)
                if o.shape != t.shape:
                    raise ValueError("out[%d] has another shape than tensors[%d]" % (i, i))
    l = lib()
    with _On(device) as on:
        norm = torch.empty((), dtype=torch.float32, device=device)
        x = (C.c_void_p * n)(*[t.data_ptr() for t in tensors])
        y = None if outs is None else (C.c_void_p * n)(*[t.data_ptr() for t in outs])
        counts = (C.c_int64 * n)(*[t.numel() for t in tensors])
        kinds = (C.c_int32 * n)(*[_DTYPES[t.dtype] for t in tensors])
        need = C.c_int64()
        _check(l.lfm_ops_clip_workspace(C.c_int64(n), counts, C.byref(need)))
        ws = on.scratch(need.value)
        _check(l.lfm_ops_clip_global_norm(C.c_int64(n), x, y, counts, kinds, C.c_double(max_norm),
                                          C.c_void_p(norm.data_ptr()), C.c_void_p(ws.data_ptr()), need,
                                          C.c_void_p(on.stream)))
    return norm


def global_norm(tensors):
    """sqrt of the sum of the squares of all elements of all tensors (summed in float64), a float32 scalar tensor."""
    return _clip(tensors, 0.0, None, False)


def clip_global_norm(tensors, max_norm, out=None):
    """Scales all tensors by min(1, max_norm / norm), norm = global_norm(tensors), in place or into the tensors of `out`,
    and returns the norm.  A norm that is not finite leaves the values unscaled: look at the returned norm."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    return _clip(tensors, max_norm, out, True)
