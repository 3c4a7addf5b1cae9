"""Operators of a full-softmax training step on tensors that live on the GPU (include/lfm_ops.h).

`LightFM(loss="softmax")` runs these kernels on its own tables; a model of the caller's that is trained with the softmax
over the whole catalogue -- a session or sequence recommender on top of the same item tables -- needs them on device
memory, between the layers of its own program.  They take and return torch tensors of one GPU:

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
autograd history (a training loop calls the gradient functions, or wraps them in its own `autograd.Function`), and warn
where a tensor requires a gradient and gradients are being recorded.

Wrong arguments raise ValueError / TypeError like the rest of the package.  There is no CPU fallback.
"""
import ctypes as C
import importlib.machinery
import importlib.util
import os

import torch

from . import _native as N

__all__ = ["softmax_loss", "softmax_loss_grad", "embedding_lookup", "embedding_lookup_grad", "global_norm",
           "clip_global_norm"]

LIB_PATH = os.path.join(os.path.dirname(N.LIB_PATH), "liblfm_ops.so")
BINDING_PATH = os.path.join(os.path.dirname(N.LIB_PATH), "_torch_ops.so")

# every symbol include/lfm_ops.h declares (tests check the .so exports them all)
EXPORTS = ("lfm_ops_last_error", "lfm_ops_softmax_workspace", "lfm_ops_softmax_loss", "lfm_ops_softmax_loss_grad",
           "lfm_ops_embedding_lookup", "lfm_ops_embedding_grad_workspace", "lfm_ops_embedding_lookup_grad",
           "lfm_ops_clip_workspace", "lfm_ops_clip_global_norm")

_lib = None


def lib():
    """liblfm_ops.so as a ctypes library, for callers of its C ABI without torch tensors; bound to the HIP runtime that torch
    uses.  Raises HipBackendError if it has not been built."""
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


class _Binding(object):
    """csrc/torch_ops.cpp, loaded with the first call."""

    def __getattr__(self, name):
        lib()
        if not os.path.exists(BINDING_PATH):
            raise N.HipBackendError("%s not found: build it with `python -m lightfm_amd.build`" % BINDING_PATH)
        loader = importlib.machinery.ExtensionFileLoader("_torch_ops", BINDING_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_torch_ops", loader))
        loader.exec_module(module)
        global _ops
        _ops = module
        return getattr(module, name)


_ops = _Binding()


def softmax_loss(hidden, table, targets, bias=None, weights=None):
    """Cross entropy of every row of `hidden` [rows, d] against all rows of `table` [vocab, d]: scores
    s = hidden table^T + bias, lse = log sum exp s, loss = weights * (lse - s[target]).  Returns (loss, lse), float32
    [rows]; a row whose target is not in [0, vocab) has loss 0.  bias [vocab] / weights [rows] are float32; a bias of
    -inf takes an item out of the softmax, whatever its row holds (as a target, its loss is infinite).  The scores are never
    kept.  float32 operands are multiplied with 22 bits and a floor of 2^-39 of the largest magnitude of hidden or table."""
    return _ops.softmax(hidden, table, targets, bias, weights, False)


def softmax_loss_grad(hidden, table, targets, bias=None, weights=None):
    """softmax_loss with the gradients of the SUM of the losses: (loss, lse, d_hidden, d_table, d_bias); d_bias is None
    without a bias.  For the mean, hand in weights of 1 / rows.  Gradients have the type of hidden / table.  An item that a
    bias of -inf takes out has a zero gradient but where it is a target: there the probability is 0 and the gradients follow the
    formula (elements of its row that are not finite count as 0)."""
    return _ops.softmax(hidden, table, targets, bias, weights, True)


def embedding_lookup(table, ids, indptr=None, values=None, scale=1.0):
    """Rows of `table` [vocab, d] times `scale`: out[r] = scale * table[ids[r]], or, with `indptr` [rows + 1] (CSR bags, as
    in a LightFM feature matrix), out[r] = scale * sum_j values[j] * table[ids[j]] over bag r.  values default to 1.
    Sums are float32 in the order of the bag; out has the type of table."""
    return _ops.lookup(table, ids, indptr, values, scale, -1)


def embedding_lookup_grad(d_out, ids, n_rows, indptr=None, values=None, scale=1.0):
    """Gradient of embedding_lookup with respect to its table of `n_rows` rows: d_table[v] = scale * sum of values[j] *
    d_out[r] over the places where ids[j] == v.  The ids are sorted and each row is summed in float32 in the order of
    their positions (no atomics: the same bits every time).  d_table is dense, of the type of d_out."""
    if n_rows < 1:
        raise ValueError("n_rows must be positive")
    return _ops.lookup(d_out, ids, indptr, values, scale, n_rows)


def global_norm(tensors):
    """sqrt of the sum of the squares of all elements of all tensors (a list or tuple), summed in float64; a float32 scalar
    tensor."""
    return _ops.clip(tensors, 0.0, None)


def clip_global_norm(tensors, max_norm, out=None):
    """Scales all tensors (a list or tuple) by min(1, max_norm / norm), norm = global_norm(tensors), in place or into the
    tensors of `out`, and returns the norm.  Where an element is not finite the norm is not either and the values are left
    unscaled: look at the returned norm (a finite norm beyond float32 is returned as infinite, and scales the values).  A
    tensor that is written overlaps no other one (ValueError)."""
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    return _ops.clip(tensors, max_norm, tensors if out is None else out)
