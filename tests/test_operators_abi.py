"""CPU-side checks of the device-memory operators: liblfm_ops.so exports what include/lfm_ops.h declares, the ctypes
structures have its layout, and wrong arguments are refused on the host before anything could be launched."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class LfmSoftmaxArgs(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("hidden", "table", "targets", "bias", "weights", "loss", "lse", "d_hidden",
                                           "d_table", "d_bias")]
                + [(n, C.c_int64) for n in ("rows", "vocab", "hidden_stride", "table_stride")]
                + [(n, C.c_int32) for n in ("d", "dtype", "id_bytes", "reserved")])


class LfmLookupArgs(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("table", "ids", "indptr", "values", "out", "d_out")]
                + [(n, C.c_int64) for n in ("rows", "vocab", "nnz", "table_stride", "d_out_stride")]
                + [(n, C.c_int32) for n in ("d", "dtype", "id_bytes")] + [("scale", C.c_float)])


@pytest.fixture(scope="module")
def ops():
    from lightfm_amd import build
    if not os.path.exists(build.OPS_LIB):
        build.build()
    from lightfm_amd import operators
    operators.lib()
    return operators


def _header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "lfm_ops.h")).read(), flags=re.S)


def test_library_exports_every_declared_symbol(ops):
    declared = set(re.findall(r"\b(lfm_ops_[a-z_0-9]+)\s*\(", _header()))
    assert declared and declared == set(ops.EXPORTS)
    for name in declared:
        assert hasattr(ops.lib(), name), name


def test_struct_layouts_match_header(ops, tmp_path):
    mirror = {"lfm_softmax_args": LfmSoftmaxArgs, "lfm_lookup_args": LfmLookupArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "lfm_ops.h"', "int main(void) {"]
    for struct, t in mirror.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (struct, struct))
        for field, _ in t._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (struct, field, struct, field))
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "probe")
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)])
    for line in subprocess.check_output([exe]).decode().splitlines():
        key, value = line.split()
        if "." in key:
            struct, field = key.split(".")
            assert getattr(mirror[struct], field).offset == int(value), key
        else:
            assert C.sizeof(mirror[key]) == int(value), key


def _softmax_args(ops, **kw):
    fake = 1 << 20  # an address that is never followed: every call below is refused on the host
    values = dict(hidden=fake, table=fake, targets=fake, bias=None, weights=None, loss=fake, lse=fake, d_hidden=fake,
                  d_table=fake, d_bias=None, rows=4, vocab=8, hidden_stride=16, table_stride=16, d=16, dtype=0,
                  id_bytes=4, reserved=0)
    values.update(kw)
    return LfmSoftmaxArgs(*[values[n] for n, _ in LfmSoftmaxArgs._fields_])


@pytest.mark.parametrize("wrong, code", [
    (dict(rows=-1), -1), (dict(vocab=0), -1), (dict(d=0), -1), (dict(d=1025), -5), (dict(dtype=3), -1),
    (dict(id_bytes=2), -1), (dict(hidden_stride=15), -1), (dict(table_stride=15), -1), (dict(hidden=None), -1),
    (dict(table=None), -1), (dict(targets=None), -1), (dict(loss=None), -1), (dict(d_hidden=None), -1),
    (dict(d_table=None), -1)])
def test_softmax_refusals(ops, wrong, code):
    a = _softmax_args(ops, **wrong)
    rc = ops.lib().lfm_ops_softmax_loss_grad(C.byref(a), C.c_void_p(1 << 20), C.c_int64(1 << 40), None)
    assert rc == code and ops.lib().lfm_ops_last_error()


def test_workspaces_are_checked(ops):
    need = C.c_int64()
    assert ops.lib().lfm_ops_softmax_workspace(C.c_int64(4), C.c_int64(8), 16, 0, 1, C.byref(need)) == 0
    a = _softmax_args(ops)
    call = ops.lib().lfm_ops_softmax_loss_grad
    assert call(C.byref(a), C.c_void_p(1 << 20), C.c_int64(need.value - 1), None) == -1
    assert call(C.byref(a), C.c_void_p((1 << 20) + 64), need, None) == -1
    assert call(C.byref(a), None, need, None) == -1
    assert call(None, C.c_void_p(1 << 20), need, None) == -1


def test_workspace_sizes_hold_at_the_limits(ops):
    """No overflow on the way to the size, and it grows with the arguments."""
    l, need = ops.lib(), C.c_int64()
    last = 0
    for rows, vocab in ((1, 1), (1 << 10, 1 << 15), (1 << 20, 1 << 24)):
        assert l.lfm_ops_softmax_workspace(C.c_int64(rows), C.c_int64(vocab), 128, 0, 1, C.byref(need)) == 0
        assert need.value >= last
        last = need.value
    assert l.lfm_ops_softmax_workspace(C.c_int64(1 << 31), C.c_int64(8), 16, 0, 1, C.byref(need)) == -1
    assert l.lfm_ops_embedding_grad_workspace(C.c_int64(1 << 20), C.c_int64((1 << 31) - 1), C.c_int64(1 << 20), 64, 0, C.byref(need)) == 0
    assert need.value >= (1 << 20) * 16
    assert l.lfm_ops_embedding_grad_workspace(C.c_int64(0), C.c_int64(5), C.c_int64(0), 64, 0, C.byref(need)) == 0
    assert l.lfm_ops_embedding_grad_workspace(C.c_int64(1), C.c_int64(0), C.c_int64(1), 64, 0, C.byref(need)) == -1


def test_long_sweeps_use_the_whole_card(ops):
    """The parts that a call joins are as many as it has blocks, and their space shows: a step of 8192 rows has as many for 391 * 128
    items as for 301 * 128, so that the larger table needs no less space (with 128 tiles to an owner, owners with a block to
    themselves would leave a quarter of the card idle)."""
    need = C.c_int64()

    def space(rows, vocab):
        assert ops.lib().lfm_ops_softmax_workspace(C.c_int64(rows), C.c_int64(vocab), 64, 1, 1, C.byref(need)) == 0
        return need.value

    assert space(8192, 391 * 128) > space(8192, 301 * 128)
    assert space(391 * 128, 26744) > space(301 * 128, 26744)


def _lookup_args(ops, **kw):
    fake = 1 << 20
    values = dict(table=fake, ids=fake, indptr=None, values=None, out=fake, d_out=fake, rows=4, vocab=8, nnz=4,
                  table_stride=16, d_out_stride=16, d=16, dtype=0, id_bytes=4, scale=1.0)
    values.update(kw)
    return LfmLookupArgs(*[values[n] for n, _ in LfmLookupArgs._fields_])


@pytest.mark.parametrize("wrong", [
    dict(rows=-1), dict(nnz=-1), dict(nnz=5), dict(vocab=0), dict(d=0), dict(d=65537), dict(dtype=7), dict(id_bytes=1),
    dict(table_stride=3), dict(d_out_stride=3), dict(values=1 << 20), dict(indptr=1 << 20, rows=0), dict(ids=None),
    dict(out=None)])
def test_lookup_refusals(ops, wrong):
    a = _lookup_args(ops, **wrong)
    if "d_out_stride" not in wrong:
        assert ops.lib().lfm_ops_embedding_lookup(C.byref(a), None) == -1
    if "table_stride" not in wrong:
        assert ops.lib().lfm_ops_embedding_lookup_grad(C.byref(a), C.c_void_p(1 << 20), C.c_int64(1 << 40), None) == -1


def test_lookup_grad_needs_an_aligned_output_and_space(ops):
    call = ops.lib().lfm_ops_embedding_lookup_grad
    assert call(C.byref(_lookup_args(ops, out=(1 << 20) + 8)), C.c_void_p(1 << 20), C.c_int64(1 << 40), None) == -1
    assert call(C.byref(_lookup_args(ops)), C.c_void_p(1 << 20), C.c_int64(0), None) == -1


def test_clip_refusals(ops):
    l = ops.lib()
    counts, kinds = (C.c_int64 * 2)(5, 7), (C.c_int32 * 2)(0, 1)
    x = (C.c_void_p * 2)(1 << 20, 1 << 21)
    ws, much, norm = C.c_void_p(1 << 20), C.c_int64(1 << 30), C.c_void_p(1 << 22)

    def call(n=2, x=x, y=x, counts=counts, kinds=kinds, top=1.0, norm=norm, ws=ws, have=much):
        return l.lfm_ops_clip_global_norm(C.c_int64(n), x, y, counts, kinds, C.c_double(top), norm, ws, have, None)

    assert call(n=-1) == -1
    assert call(counts=(C.c_int64 * 2)(5, -7)) == -1
    assert call(kinds=(C.c_int32 * 2)(0, 9)) == -1
    assert call(x=(C.c_void_p * 2)(1 << 20, None)) == -1
    assert call(y=(C.c_void_p * 2)(1 << 20, None)) == -1
    assert call(top=-1.0) == -1 and call(top=float("nan")) == -1
    assert call(norm=None) == -1
    assert call(have=C.c_int64(0)) == -1
    need = C.c_int64()
    assert l.lfm_ops_clip_workspace(C.c_int64(2), counts, None) == -1
    assert l.lfm_ops_clip_workspace(C.c_int64(2), counts, C.byref(need)) == 0 and need.value >= 16


def test_python_layer_refuses_wrong_tensors(ops):
    """Types, shapes and places, on CPU tensors (which are themselves refused: there is no CPU fallback)."""
    import torch
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError):
        ops.softmax_loss(x.numpy(), w, t)
    with pytest.raises(ValueError, match="dtype"):
        ops.softmax_loss(x.double(), w.double(), t)
    with pytest.raises(ValueError, match="dimensions"):
        ops.softmax_loss(x[0], w, t)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.softmax_loss(x, w, t)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.embedding_lookup(w, t)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.embedding_lookup_grad(x, t, 5)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.clip_global_norm([x], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_global_norm([x], -1.0)
    with pytest.raises(ValueError, match="no tensors"):
        ops.global_norm([])


def test_python_layer_warns_where_autograd_would_be_lost(ops):
    """A tensor that requires a gradient, while gradients are recorded: the results carry none.  (The calls end at the place
    of the tensors.)"""
    import warnings

    import torch
    x, w = torch.zeros(3, 8), torch.zeros(5, 8, requires_grad=True)
    t = torch.zeros(3, dtype=torch.int64)
    calls = [lambda w: ops.softmax_loss(x, w, t), lambda w: ops.softmax_loss_grad(x, w, t), lambda w: ops.embedding_lookup(w, t),
             lambda w: ops.global_norm([w]), lambda w: ops.clip_global_norm([w], 1.0)]
    for call in calls:
        with pytest.warns(UserWarning, match="does not record"), pytest.raises(ValueError, match="no CPU fallback"):
            call(w)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            with pytest.raises(UserWarning):
                call(w)
            with torch.no_grad(), pytest.raises(ValueError, match="no CPU fallback"):
                call(w)
            with pytest.raises(ValueError, match="no CPU fallback"):
                call(w.detach())
