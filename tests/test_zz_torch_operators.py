"""The device-memory operators (lightfm_amd.operators) on the GPU against plain 64-bit restatements of their formulas.

Tolerances are bounds, not samples.  u(t) = finfo(t).eps / 2 is a rounding's largest relative error.  With A = |x| |w|^T
a score's error is at most d u32 A (accumulation) + 2^-20 A (float32 operands are multiplied as two 11-bit halves each:
an operand is off by 2^-22 at most and the product of the low halves, 2^-22, is left out; half-precision operands are
multiplied exactly) + 4 u32 (|s| + |b|) (the additions and the scaling to base 2).  A sum of n positive terms is off by
n u32, relatively; exp2 and log2 by a few units of the last place.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def env():
    import torch
    if not torch.cuda.is_available():
        from lightfm_amd import _native
        assert _native.device_count() == 0, "torch does not see the GPU that the library sees"
        pytest.skip("no GPU")
    from lightfm_amd import operators
    return torch, operators


DTYPE = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def unit(torch, dtype):
    return torch.finfo(dtype).eps / 2


def make(torch, rows, vocab, d, dtype, seed=0, bias=True, weights=True, ids="int64", size=None, ignored=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000 + seed)
    dt = getattr(torch, DTYPE[dtype])
    size = math.sqrt(2.0 / math.sqrt(d)) if size is None else size
    x = (torch.randn(rows, d, generator=g, device="cuda") * size).to(dt)
    w = (torch.randn(vocab, d, generator=g, device="cuda") * size).to(dt)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if ignored and rows > 4:
        t[1] = -1
        t[rows // 2] = vocab
        t[rows - 1] = -7
    b = torch.randn(vocab, generator=g, device="cuda") if bias else None
    k = torch.rand(rows, generator=g, device="cuda") + 0.1 if weights else None
    return x, w, t.to(getattr(torch, ids)), b, k


def reference(torch, x, w, t, b, k):
    """(values, bounds): loss, lse, d_hidden, d_table, d_bias in 64 bits and how far a result may be off, derived as in the
    module's docstring."""
    dt = x.dtype
    u, d = unit(torch, dt), x.shape[1]
    has = (t >= 0) & (t < w.shape[0])
    t = torch.where(has, t.long(), torch.zeros_like(t).long())
    live = has[:, None]
    xx = x.double()
    ww = w.double()
    bb = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if b is None else b.double()
    g = has.double() if k is None else torch.where(has, k.double(), torch.zeros_like(k).double())
    s = xx @ ww.t() + bb
    big = torch.nan_to_num(s.abs(), posinf=0.0) + torch.nan_to_num(bb.abs(), posinf=0.0)
    ds = (d * U32 + 2.0 ** -20) * (xx.abs() @ ww.abs().t()) + 4 * U32 * big
    lse = torch.logsumexp(s, 1)
    n_sum = (w.shape[0] + 64) * U32
    dmax = ds.max(1).values
    dlse = dmax + n_sum + 8 * U32 * (1 + torch.nan_to_num(lse.abs(), posinf=0.0))
    st = s.gather(1, t[:, None]).squeeze(1)
    loss = torch.where(has, g * (lse - st), torch.zeros_like(lse))
    dloss = g.abs() * (dlse + ds.gather(1, t[:, None]).squeeze(1) + 8 * U32 * torch.nan_to_num(st.abs(), posinf=0.0)) + 8 * U32 * torch.nan_to_num(loss.abs(), posinf=0.0)
    p = torch.exp(s - lse[:, None])
    dp = p * (ds + dlse[:, None] + 16 * U32)          # of the float32 value
    hot = torch.zeros_like(p)
    hot[torch.arange(x.shape[0], device=x.device), t] = 1.0
    q = torch.where(live, g[:, None] * (p - hot), torch.zeros_like(p))
    half = u if dt != torch.float32 else 2.0 ** -21   # what the value loses on its way into the matrix product
    e1 = g[:, None].abs() * (dp + half * p)
    e2 = g[:, None].abs() * dp + (half + 2 * U32) * q.abs() + 2.0 ** -26 * g.abs().max()
    e1, e2 = (torch.where(live, e, torch.zeros_like(e)) for e in (e1, e2))
    xz = torch.where(live, xx, torch.zeros_like(xx))
    acc = U32 * max(w.shape[0], x.shape[0])           # accumulation of the second product
    dx, dw, db = q @ ww, q.t() @ xz, q.sum(0)
    tx = e1 @ ww.abs() + (acc + 2.0 ** -20) * (g[:, None].abs() * (torch.where(live, p, torch.zeros_like(p)) + hot)) @ ww.abs() + 2 * u * dx.abs()
    tw = e2.t() @ xz.abs() + (acc + 2.0 ** -20) * (q.abs().t() @ xz.abs()) + 2 * u * dw.abs()
    tb = (g[:, None].abs() * dp).sum(0) * live.any() + (x.shape[0] + 64) * U32 * q.abs().sum(0) + 4 * U32 * hot.t() @ g.abs()
    tiny = torch.finfo(dt).tiny if dt != torch.float16 else 2.0 ** -24
    return ((loss, lse, dx, dw, db), (dloss, dlse, tx + tiny, tw + tiny, tb + 1e-30))


def near(torch, got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~((off <= bound) | same)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its bound, e.g. %r against %r (bound %r)" % (
        what, int(bad.sum()), bad.numel(), float((off / bound)[bad].max()), got[bad][:3].tolist(), want[bad][:3].tolist(), bound.expand_as(off)[bad][:3].tolist())


def check_softmax(env, x, w, t, b, k):
    torch, ops = env
    (loss, lse, dx, dw, db), (tl, te, tx, tw, tb) = reference(torch, x, w, t, b, k)
    got = ops.softmax_loss(x, w, t, bias=b, weights=k)
    near(torch, got[0], loss, tl, "loss")
    near(torch, got[1], lse, te, "lse")
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    near(torch, got[0], loss, tl, "loss with gradient")
    near(torch, got[1], lse, te, "lse with gradient")
    near(torch, got[2], dx, tx, "d_hidden")
    near(torch, got[3], dw, tw, "d_table")
    if b is None:
        assert got[4] is None
    else:
        near(torch, got[4], db, tb, "d_bias")
    assert got[2].dtype == x.dtype and got[3].dtype == w.dtype
    return got


SIZES = [(1, 1, 1), (1, 2, 3), (2, 1682, 10), (5, 64, 16), (33, 257, 31), (64, 1000, 64), (65, 1023, 65), (130, 999, 100),
         (129, 515, 128), (200, 300, 200), (31, 2050, 256), (257, 129, 33), (1000, 31, 96), (40, 700, 300), (20, 500, 512),
         (17, 300, 1000), (300, 40, 1024), (1, 5000, 64), (2, 4097, 129), (16, 3001, 17)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, vocab, d", SIZES)
def test_softmax_sizes(env, rows, vocab, d, dtype):
    torch, ops = env
    check_softmax(env, *make(torch, rows, vocab, d, dtype, seed=rows + vocab))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias, weights, ids", [(False, False, "int32"), (True, False, "int64"), (False, True, "int32")])
@pytest.mark.parametrize("rows, vocab, d", [(70, 333, 48), (3, 900, 64), (150, 3500, 20)])
def test_softmax_variants(env, rows, vocab, d, dtype, bias, weights, ids):
    torch, ops = env
    check_softmax(env, *make(torch, rows, vocab, d, dtype, seed=3, bias=bias, weights=weights, ids=ids))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_softmax_many_rows_and_a_large_vocabulary(env, dtype):
    torch, ops = env
    check_softmax(env, *make(torch, 3000, 130, 64, dtype, seed=5))
    check_softmax(env, *make(torch, 140, 20011, 72, dtype, seed=6))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_softmax_strided_rows_and_odd_addresses(env, dtype):
    torch, ops = env
    x, w, t, b, k = make(torch, 77, 401, 61, dtype, seed=9)
    x2 = torch.full((77, 100), float("nan"), dtype=x.dtype, device="cuda")[:, 3:64]
    w2 = torch.full((401, 67), float("nan"), dtype=x.dtype, device="cuda")[:, 5:66]
    x2.copy_(x)
    w2.copy_(w)
    assert not x2.is_contiguous() and not w2.is_contiguous()
    a, c = check_softmax(env, x, w, t, b, k), check_softmax(env, x2, w2, t, b, k)
    for i, j in zip(a, c):
        assert torch.equal(i, j)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 90])
def test_softmax_masked_items(env, dtype, rows):
    """A bias of -inf takes items out: their gradient is zero unless they are targets; a target that is out has an
    infinite loss.  A bias of float32's lowest value is a finite score that only counts where nothing else does."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 500, 40, dtype, seed=11, ignored=False)
    b[100:400] = -math.inf
    b[400:450] = torch.finfo(torch.float32).min
    t[t >= 100] = 7
    got = check_softmax(env, x, w, t, b, k)
    assert (got[3][100:450] == 0).all() and (got[4][100:450] == 0).all()
    t[2] = 200
    loss = ops.softmax_loss(x, w, t, bias=b, weights=k)[0]
    assert math.isinf(float(loss[2])) and float(loss[2]) > 0
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    assert math.isinf(float(got[0][2])) and all(torch.isfinite(o).all() for o in got[1:])
    (_, _, dx, dw, db), (_, _, tx, tw, tb) = reference(torch, x, w, t, b, k)
    near(torch, got[2], dx, tx, "d_hidden")
    near(torch, got[3], dw, tw, "d_table")
    near(torch, got[4], db, tb, "d_bias")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [2, 40])
def test_softmax_nothing_left(env, dtype, rows):
    """Every item out: lse is -inf, the loss infinite, the gradient only what the target itself contributes."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 300, 24, dtype, seed=12, ignored=False)
    b[:] = -math.inf
    loss, lse, dx, dw, db = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    assert (lse == -math.inf).all() and (loss == math.inf).all()
    wt = -k[:, None].double() * w.double()[t]
    near(torch, dx, wt, (unit(torch, x.dtype) * 2 + 2.0 ** -20) * wt.abs() + 2.0 ** -24, "d_hidden")
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    want = torch.zeros(300, dtype=torch.float64, device="cuda").index_add_(0, t.long(), -k.double())
    near(torch, db, want, (rows + 4) * U32 * want.abs() + 1e-30, "d_bias")
    b[:] = torch.finfo(torch.float32).min
    loss, lse = ops.softmax_loss(x, w, t, bias=b, weights=k)
    assert torch.isfinite(loss).all()
    near(torch, lse, torch.full_like(lse, torch.finfo(torch.float32).min).double(), torch.tensor(2.0 ** 105, device="cuda").double(), "lse")


@pytest.mark.parametrize("d", [1, 50, 51, 64, 257, 300])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
def test_softmax_few_float32_rows(env, rows, d):
    check_softmax(env, *make(env[0], rows, 3001, d, "f32", seed=rows, ignored=rows > 4))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, d", [(2, 98), (31, 128), (32, 65), (33, 200), (64, 96), (65, 128), (64, 32), (20, 256)])
def test_softmax_one_tile_of_rows(env, rows, d, dtype):
    """At and around the number of rows that is one tile of the table's sweep (64, or 32 for wide rows); the table ends inside
    the last owner of 128."""
    check_softmax(env, *make(env[0], rows, 9011, d, dtype, seed=rows + d))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_softmax_offsets_past_32_bits(env, dtype):
    """A table of more than 2^32 elements: scores, gradients and targets at both ends of it."""
    torch, ops = env
    vocab, d, rows, step = 67500001, 64, 9, 1 << 22
    x, _, _, _, k = make(torch, rows, 8, d, dtype, seed=15, ignored=False)
    w = torch.empty(vocab, d, dtype=x.dtype, device="cuda").normal_(0.0, 0.3)
    t = torch.tensor([0, 1, 33554432, 67108863, 67108864, vocab - 1, vocab - 2, vocab, -1], device="cuda")
    has = (t >= 0) & (t < vocab)
    g = torch.where(has, k, torch.zeros_like(k)).double()
    xx = x.double()
    lse = torch.full((rows,), -math.inf, dtype=torch.float64, device="cuda")
    for lo in range(0, vocab, step):
        lse = torch.logaddexp(lse, torch.logsumexp(xx @ w[lo:lo + step].double().t(), 1))
    dx = torch.zeros(rows, d, dtype=torch.float64, device="cuda")
    for lo in range(0, vocab, step):
        ww = w[lo:lo + step].double()
        dx += torch.exp(xx @ ww.t() - lse[:, None]) @ ww
    wt = w[t.clamp(0, vocab - 1)].double()
    loss = torch.where(has, g * (lse - (xx * wt).sum(1)), torch.zeros_like(lse))
    dx = g[:, None] * (dx - wt)
    got = ops.softmax_loss_grad(x, w, t, weights=k)
    # scores are good to 2^-18 (2^-20 of |x||w| < 3 and less); the float32 sums over 2^26 items are joined from some hundred parts
    # of tiles that are added in pairs: 2^-14 is far above their rounding and far below a row that is read in a wrong place
    near(torch, got[1], lse, 2.0 ** -14 * lse.abs(), "lse")
    near(torch, got[0], loss, 2.0 ** -14 * (lse.abs() + 1), "loss")
    near(torch, got[2], dx, (2 * unit(torch, x.dtype) + 2.0 ** -14) * (dx.abs() + g[:, None]), "d_hidden")
    at = torch.cat([t[has], torch.tensor([2, 33554431, 33554433, 50000000, 67108865, vocab - 3], device="cuda")])
    q = torch.exp(xx @ w[at].double().t() - lse[:, None])
    q = g[:, None] * (q - (t[:, None] == at[None, :]).double())
    dw = q.t() @ torch.where(has[:, None], xx, torch.zeros_like(xx))
    # float32: q is multiplied by 2^(14 - e), 2^e >= the largest weight > 2^(e - 1), and cut into two float16, the second to
    # nearest: where that is subnormal (steps of 2^-24) q is off by 2^-25 2^(e - 14) <= 2^-38 of the largest weight
    floor = 2.0 ** -38 * float(g.max()) if dtype == "f32" else 0.0
    near(torch, got[3][at], dw, (4 * unit(torch, x.dtype) + 2.0 ** -14) * (q.abs().t() @ xx.abs()) + floor * torch.where(has[:, None], xx.abs(), torch.zeros_like(xx)).sum(0) + 1e-30, "d_table")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, d", [(2, 64), (70, 64), (70, 50), (33, 300)])
def test_softmax_removed_items_hold_anything(env, dtype, rows, d):
    """NaN, infinities and the type's largest values in the rows of removed items: the results are those of zeros there,
    bit for bit (in place, packed, in chunks of columns, and with few rows)."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 420, d, dtype, seed=14, ignored=False)
    gone = torch.zeros(420, dtype=torch.bool, device="cuda")
    gone[[0, 3, 64, 65, 200, 419]] = True
    gone[300:390] = True
    t[gone[t.long()]] = 7
    b[gone] = -math.inf
    w[gone] = 0
    clean = check_softmax(env, x, w, t, b, k)
    few = ops.softmax_loss(x, w, t, bias=b, weights=k)
    w[gone] = torch.finfo(w.dtype).max
    w[3], w[64], w[65, 1], w[320:340] = float("nan"), math.inf, -math.inf, -math.inf
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    for i in range(5):
        assert torch.equal(got[i], clean[i]), i
    for one, other in zip(ops.softmax_loss(x, w, t, bias=b, weights=k), few):
        assert torch.equal(one, other)
    assert (got[3][gone] == 0).all() and (got[4][gone] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [12, 100])
def test_softmax_rows_without_target_are_not_read(env, dtype, rows):
    """NaN and infinities in rows without a target touch nothing but their own lse."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 210, 50, dtype, seed=13, ignored=False)
    out = torch.zeros(rows, dtype=torch.bool, device="cuda")
    out[[1, 5, 6, rows - 1]] = True
    t[out] = -1
    clean = ops.softmax_loss_grad(torch.where(out[:, None], torch.zeros_like(x), x), w, t, bias=b, weights=k)
    x[1], x[5], x[6], x[rows - 1, 3] = float("nan"), math.inf, -math.inf, float("nan")
    k[1], k[5] = float("nan"), math.inf
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    assert (got[0][out] == 0).all() and (got[2][out] == 0).all()
    for i in (0, 2, 3, 4):
        assert torch.equal(got[i], clean[i]), i
    assert torch.equal(got[1][~out], clean[1][~out])
    assert torch.equal(ops.softmax_loss(x, w, t, bias=b, weights=k)[0], ops.softmax_loss(torch.where(out[:, None], torch.zeros_like(x), x), w, t, bias=b, weights=k)[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_softmax_no_rows_and_only_rows_without_target(env, dtype):
    torch, ops = env
    x, w, t, b, k = make(torch, 6, 90, 33, dtype, seed=14)
    got = ops.softmax_loss_grad(x[:0], w, t[:0], bias=b, weights=k[:0])
    assert got[0].shape == (0,) and got[2].shape == (0, 33)
    assert (got[3] == 0).all() and (got[4] == 0).all() and got[3].shape == (90, 33)
    assert ops.softmax_loss(x[:0], w, t[:0])[0].shape == (0,)
    t[:] = -1
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    assert all((got[i] == 0).all() for i in (0, 2, 3, 4))
    near(torch, got[1], torch.logsumexp(x.double() @ w.double().t() + b.double(), 1), reference(torch, x, w, t, b, k)[1][1], "lse")


@pytest.mark.parametrize("size", [1e-18, 1e-3, 30.0, 1e6])
@pytest.mark.parametrize("rows", [4, 60])
def test_softmax_float32_magnitudes(env, size, rows):
    """Very small and very large float32 operands: scores from 0 to 1e13.  (The bounds scale with the scores: at 1e13 they
    allow any probability, at 30 they still tell the gradients apart.)"""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 700, 36, "f32", seed=15, size=size)
    (loss, lse, dx, dw, db), bounds = reference(torch, x, w, t, b, k)
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    assert all(torch.isfinite(o).all() for o in got)
    for name, o, want, bound in zip(("loss", "lse", "d_hidden", "d_table", "d_bias"), got, (loss, lse, dx, dw, db), bounds):
        if size <= 30.0 or name in ("loss", "lse"):
            near(torch, o, want, bound, name)


@pytest.mark.parametrize("rows", [5, 50])
def test_softmax_float32_operands_of_unlike_size(env, rows):
    """Tiny hidden rows against a large table, rows of very unlike size in one table."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 600, 40, "f32", seed=16)
    check_softmax(env, x * 1e-12, w * 1e12, t, b, k)
    w[::3] *= 1e-4
    x[::2] *= 1e-3
    check_softmax(env, x, w, t, b, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_softmax_weights_of_unlike_size_and_sign(env, dtype):
    torch, ops = env
    x, w, t, b, k = make(torch, 90, 333, 30, dtype, seed=17)
    k[::4] *= 1e-3
    k[::5] *= -20.0
    k[3] = 0.0
    check_softmax(env, x, w, t, b, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_softmax_same_bits_every_time(env, dtype):
    torch, ops = env
    x, w, t, b, k = make(torch, 300, 5003, 64, dtype, seed=18)
    first = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    for _ in range(3):
        for i, j in zip(first, ops.softmax_loss_grad(x, w, t, bias=b, weights=k)):
            assert torch.equal(i, j)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [6, 70])
def test_softmax_rows_that_fit_well(env, dtype, rows):
    """Targets with a probability near 1: loss and gradient are small differences and keep their relative precision (the
    target's part is formed from the sum over the OTHER items).  Bounds: a probability is off by ds + dlse as in `reference`,
    relatively; every product's operand by `half` of its own size; so all errors are relative to sums of |q|-like terms."""
    torch, ops = env
    x, w, t, b, _ = make(torch, rows, 400, 64, dtype, seed=21, weights=False, ignored=False)
    t = torch.randperm(400, device="cuda")[:rows]
    x = (w[t].double() * 0.9 + x.double() * 0.1).to(x.dtype)   # s[target] ~ 0.9 |w|^2 ~ 14, the others ~ N(0, 4)
    loss, lse, dx, dw, db = ops.softmax_loss_grad(x, w, t, bias=b)
    xx, ww = x.double(), w.double()
    s = xx @ ww.t() + b.double()
    ds = (64 * U32 + 2.0 ** -20) * (xx.abs() @ ww.abs().t()) + 8 * U32 * s.abs()
    rel = 2 * ds.max(1).values[:, None] + (400 + 128) * U32       # of exp(s - s_target) and of sums of them
    st = s.gather(1, t[:, None])
    e = torch.exp(s - st)
    e[torch.arange(rows, device="cuda"), t] = 0.0
    others = e.sum(1, keepdim=True)
    assert float(others.median()) < 0.05
    want = torch.log1p(others).squeeze(1)
    near(torch, loss, want, (rel.squeeze(1) + 8 * U32) * want, "loss")
    q, rest = e / (1 + others), others / (1 + others)
    half = 2.0 ** -21 if dtype == "f32" else unit(torch, x.dtype)
    u = 2 * unit(torch, x.dtype)
    gx = q @ ww - rest * ww[t]
    near(torch, dx, gx, (2 * rel + half + 2.0 ** -19) * (q @ ww.abs() + rest * ww[t].abs()) + u * gx.abs() + 2.0 ** -24, "d_hidden")
    hot = torch.zeros_like(q)
    hot[torch.arange(rows, device="cuda"), t] = 1.0
    gw = q.t() @ xx - hot.t() @ (rest * xx)
    near(torch, dw, gw, ((2 * rel + half + 2.0 ** -19) * q).t() @ xx.abs() + hot.t() @ ((2 * rel + half) * rest * xx.abs()) + u * gw.abs() + 2.0 ** -24, "d_table")
    gb = q.sum(0) - (hot * rest).sum(0)
    near(torch, db, gb, ((2 * rel + 128 * U32) * (q + hot * rest)).sum(0) + 1e-30, "d_bias")


def test_softmax_gradient_against_differences(env):
    """sum(loss) along random directions: (L(+h) - L(-h)) / 2h, from a 64-bit restatement of the LOSS alone, against the
    kernel's gradients.  The difference's own error: h^2 / 6 times the third derivative along the direction, at most
    sum_n 2 max_v |ds_nv|^3 <= 2 rows D^3 with D the largest change of a score, and 64-bit rounding / h."""
    torch, ops = env
    x, w, t, b, k = make(torch, 25, 130, 18, "f32", seed=19)
    _, _, dx, dw, db = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    (_, _, *_), (_, _, tx, tw, tb) = reference(torch, x, w, t, b, k)
    has = (t >= 0) & (t < w.shape[0])

    def total(x, w, b):
        s = x @ w.t() + b
        each = torch.logsumexp(s, 1) - s.gather(1, t.clamp(0, w.shape[0] - 1)[:, None]).squeeze(1)
        return (each * k.double() * has).sum()

    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    h = 1e-4
    for part, grad, bound in ((0, dx, tx), (1, dw, tw), (2, db, tb)):
        at = [x.double(), w.double(), b.double()]
        u = torch.randn(at[part].shape, generator=g, device="cuda", dtype=torch.float64)
        up, down = list(at), list(at)
        up[part], down[part] = at[part] + h * u, at[part] - h * u
        slope = (total(*up) - total(*down)) / (2 * h)
        change = [lambda: u @ at[1].t(), lambda: at[0] @ u.t(), lambda: u][part]().abs().max()
        error = h * h / 6 * 2 * 25 * float(k.max()) * float(change) ** 3 + 2.0 ** -52 * 1e3 / h
        assert abs(float(slope - (grad.double() * u).sum())) <= error + float((bound * u.abs()).sum())


# ------------------------------------------------------------------ lookup ---

def bags(torch, rows, vocab, per_bag, seed, ids="int32", skew=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(77 + seed)
    if per_bag:
        lengths = torch.randint(0, 2 * per_bag + 1, (rows,), generator=g, device="cuda")
        indptr = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        indptr[1:] = torch.cumsum(lengths, 0)
        nnz = int(indptr[-1])
        values = torch.randn(nnz, generator=g, device="cuda")
    else:
        indptr = values = None
        nnz = rows
    r = torch.rand(nnz, generator=g, device="cuda", dtype=torch.float64)
    at = (torch.exp(r * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1) if skew else (r * vocab).long().clamp_(0, vocab - 1)
    if nnz > 10:
        at[3], at[nnz // 2] = -1, vocab
    it = getattr(torch, ids)
    return at.to(it), None if indptr is None else indptr.to(it), values


def bag_rows(torch, ids, indptr):
    rows = torch.arange(ids.shape[0] if indptr is None else indptr.shape[0] - 1, device=ids.device)
    return rows if indptr is None else torch.repeat_interleave(rows, indptr.long().diff())


def check_lookup(env, table, ids, indptr, values, scale):
    torch, ops = env
    rows, d = (ids.shape[0] if indptr is None else indptr.shape[0] - 1), table.shape[1]
    ok = (ids >= 0) & (ids < table.shape[0])
    picked = torch.where(ok[:, None], table.double()[ids.long().clamp(0, table.shape[0] - 1)], torch.zeros((), dtype=torch.float64, device="cuda"))
    if values is not None:
        picked = picked * values.double()[:, None]
    where = bag_rows(torch, ids, indptr)
    want = torch.zeros(rows, d, dtype=torch.float64, device="cuda").index_add_(0, where, picked) * scale
    mass = torch.zeros(rows, d, dtype=torch.float64, device="cuda").index_add_(0, where, picked.abs()) * abs(scale)
    longest = 1 if indptr is None else int(indptr.long().diff().max()) if rows else 1
    got = ops.embedding_lookup(table, ids, indptr=indptr, values=values, scale=scale)
    assert got.dtype == table.dtype
    near(torch, got, want, (longest + 2) * U32 * mass + unit(torch, table.dtype) * want.abs() * (1 + 2.0 ** -7) + torch.finfo(torch.float32).tiny + (2.0 ** -25 if table.dtype == torch.float16 else 0.0), "lookup")


def check_lookup_grad(env, d_out, ids, vocab, indptr, values, scale):
    torch, ops = env
    d = d_out.shape[1]
    ok = (ids >= 0) & (ids < vocab)
    each = torch.where(ok[:, None], d_out.double()[bag_rows(torch, ids, indptr)], torch.zeros((), dtype=torch.float64, device="cuda"))
    if values is not None:
        each = each * values.double()[:, None]
    to = ids.long().clamp(0, vocab - 1)
    want = torch.zeros(vocab, d, dtype=torch.float64, device="cuda").index_add_(0, to, each) * scale
    mass = torch.zeros(vocab, d, dtype=torch.float64, device="cuda").index_add_(0, to, each.abs()) * abs(scale)
    count = int(torch.bincount(to, minlength=1).max()) if to.numel() else 1
    got = ops.embedding_lookup_grad(d_out, ids, vocab, indptr=indptr, values=values, scale=scale)
    assert got.dtype == d_out.dtype
    near(torch, got, want, (count + 3) * U32 * mass + unit(torch, d_out.dtype) * want.abs() * (1 + 2.0 ** -7) + torch.finfo(torch.float32).tiny + (2.0 ** -25 if d_out.dtype == torch.float16 else 0.0), "lookup gradient")
    assert (got[(mass == 0).all(1)] == 0).all()
    return got


LOOKUPS = [(1, 1, 1), (1, 50, 64), (3, 7, 5), (63, 100, 10), (500, 37, 33), (1000, 3000, 64), (4097, 501, 100), (700, 90000, 128),
           (2000, 2047, 256), (300, 2048, 300), (129, 5000000, 8), (50000, 11, 16), (9000, 40000, 1030)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per_bag", [0, 5])
@pytest.mark.parametrize("rows, vocab, d", LOOKUPS)
def test_lookup_and_gradient(env, rows, vocab, d, per_bag, dtype):
    torch, ops = env
    dt = getattr(torch, DTYPE[dtype])
    ids, indptr, values = bags(torch, rows, vocab, per_bag, seed=d, ids="int32" if d % 2 else "int64")
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    check_lookup(env, torch.randn(vocab, d, generator=g, device="cuda").to(dt), ids, indptr, values, 0.75)
    first = check_lookup_grad(env, torch.randn(rows, d, generator=g, device="cuda").to(dt), ids, vocab, indptr, values, 0.75)
    assert first.shape == (vocab, d)


def test_lookup_long_lists(env):
    """Several sort digits, several pieces per sort block, runs over thousands of chunks."""
    torch, ops = env
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    for rows, vocab, d, skew in ((700001, 300007, 12, True), (600000, 3, 20, False), (1000003, 5000011, 4, False)):
        ids, _, _ = bags(torch, rows, vocab, 0, seed=rows, skew=skew)
        x = torch.randn(rows, d, generator=g, device="cuda")
        first = check_lookup_grad(env, x, ids, vocab, None, None, 1.0)
        assert torch.equal(first, ops.embedding_lookup_grad(x, ids, vocab))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab, d", [(4096, 3, 70), (4097, 3, 70), (65536, 900, 131), (65537, 7, 34), (150001, 20011, 6), (200001, 40, 257)])
def test_lookup_gradient_at_the_lengths_where_the_form_changes(env, rows, vocab, d, dtype):
    torch, ops = env
    ids, _, _ = bags(torch, rows, vocab, 0, seed=rows + d, skew=True)
    x = torch.randn(rows, d, device="cuda").to(getattr(torch, DTYPE[dtype]))
    first = check_lookup_grad(env, x, ids, vocab, None, None, 1.25)
    assert torch.equal(first, ops.embedding_lookup_grad(x, ids, vocab, scale=1.25))


def test_lookup_one_id_only_and_all_out_of_range(env):
    torch, ops = env
    x = torch.randn(5000, 24, device="cuda")
    ids = torch.full((5000,), 2, dtype=torch.int32, device="cuda")
    check_lookup_grad(env, x, ids, 5, None, None, 2.0)
    for bad in (-1, 5, 2 ** 31 - 1, -2 ** 31):
        ids[:] = bad
        assert (ops.embedding_lookup_grad(x, ids, 5) == 0).all()
        assert (ops.embedding_lookup(torch.ones(5, 24, device="cuda"), ids) == 0).all()
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 1], device="cuda")
    assert (ops.embedding_lookup(torch.ones(5, 24, device="cuda"), far) == 0).all()
    assert (ops.embedding_lookup_grad(x[:3].contiguous(), far, 5) == 0).all()


def test_lookup_empty(env):
    torch, ops = env
    w = torch.randn(9, 6, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.embedding_lookup(w, none).shape == (0, 6)
    assert (ops.embedding_lookup_grad(w[:0], none, 9) == 0).all()
    empty = torch.zeros(5, dtype=torch.int64, device="cuda")   # four empty bags
    assert (ops.embedding_lookup(w, none, indptr=empty) == 0).all()
    assert (ops.embedding_lookup_grad(torch.ones(4, 6, device="cuda"), none, 9, indptr=empty) == 0).all()
    one = torch.zeros(1, dtype=torch.int64, device="cuda")     # no bags
    assert ops.embedding_lookup(w, none, indptr=one).shape == (0, 6)
    assert (ops.embedding_lookup_grad(w[:0], none, 9, indptr=one) == 0).all()


def test_lookup_broken_indptr_stays_inside(env):
    """Extents that are not monotone or leave [0, nnz] are cut to it: no read outside, the good bags keep their sums."""
    torch, ops = env
    w = torch.randn(20, 8, device="cuda")
    ids = torch.arange(12, dtype=torch.int32, device="cuda")
    indptr = torch.tensor([0, 4, -5, 99, 12], dtype=torch.int32, device="cuda")
    out = ops.embedding_lookup(w, ids, indptr=indptr)
    assert torch.allclose(out[0], w[:4].sum(0), atol=1e-5) and torch.isfinite(out).all()
    assert torch.isfinite(ops.embedding_lookup_grad(torch.randn(4, 8, device="cuda"), ids, 20, indptr=indptr)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_lookup_strided_rows(env, dtype):
    torch, ops = env
    dt = getattr(torch, DTYPE[dtype])
    wide = torch.randn(60, 50, device="cuda").to(dt)
    for lo, hi in ((0, 16), (1, 18), (8, 40), (3, 50)):
        ids, indptr, values = bags(torch, 200, 60, 4, seed=lo)
        check_lookup(env, wide[:, lo:hi], ids, indptr, values, 1.5)
        ids, _, _ = bags(torch, 60, 30, 0, seed=lo)
        check_lookup_grad(env, wide[:, lo:hi], ids, 30, None, None, 1.5)


def test_lookup_offsets_past_32_bits(env):
    """A table of more than 2^32 elements (bytes past 2^33)."""
    torch, ops = env
    vocab, d = 70000000, 64
    w = torch.empty(vocab, d, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, 33554432, 67108864, vocab - 1, vocab], device="cuda")
    for i, at in enumerate(ids[:4].tolist()):
        w[at] = torch.arange(d, device="cuda").to(torch.bfloat16) + i
    out = ops.embedding_lookup(w, ids)
    for i in range(4):
        assert torch.equal(out[i], torch.arange(d, device="cuda").to(torch.bfloat16) + i)
    assert (out[4] == 0).all()
    del w
    x = torch.randn(5, d, device="cuda").to(torch.bfloat16)
    g = ops.embedding_lookup_grad(x, ids, vocab)
    for i, at in enumerate(ids[:4].tolist()):
        assert torch.equal(g[at], x[i])
        g[at] = 0
    assert not g.view(torch.int32).any()


def test_lookup_of_more_lanes_than_one_dimension_of_a_launch(env):
    """2^30 + 80 lanes: a launch of two rows of blocks."""
    torch, ops = env
    rows, d = (1 << 26) + 5, 128
    w = torch.randn(1009, d, device="cuda").to(torch.bfloat16)
    ids = (torch.arange(rows, device="cuda") % 1009).int()
    out = ops.embedding_lookup(w, ids)
    for lo in range(0, rows, 1 << 22):
        assert torch.equal(out[lo:lo + (1 << 22)], w[ids[lo:lo + (1 << 22)].long()]), lo


# -------------------------------------------------------------------- clip ---

def check_clip(env, tensors, max_norm, out=None):
    torch, ops = env
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    factor = min(1.0, max_norm / norm) if norm > 0 else 1.0
    want = [t.double() * factor for t in tensors]
    got_norm = ops.clip_global_norm(tensors, max_norm, out=out)
    assert got_norm.dtype == torch.float32 and got_norm.shape == ()
    assert abs(float(got_norm) - norm) <= 2 * U32 * norm
    for g, w in zip(tensors if out is None else out, want):
        near(torch, g, w, (unit(torch, g.dtype) * (1 + 2.0 ** -7) + 3 * U32) * w.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 1e-38), "clipped")


CLIPS = [[1], [0, 5], [32768, 1, 32769], [3, 100000, 7, 0, 65536], [1000] * 63, [17] * 64, [1001] * 65, [5] * 200, [5000003, 2, 300007]]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", CLIPS, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_clip(env, sizes, dtype):
    torch, ops = env
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    kinds = list(DTYPE) if dtype == "mixed" else [dtype]
    ts = [torch.randn(n, generator=g, device="cuda").to(getattr(torch, DTYPE[kinds[i % len(kinds)]])) for i, n in enumerate(sizes)]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    assert abs(float(ops.global_norm(ts)) - norm) <= 2 * U32 * norm
    out = [torch.full_like(t, 7.0) for t in ts]
    before = [t.clone() for t in ts]
    for top in (norm * 0.3, norm * 2.0, 0.0):
        check_clip(env, ts, top, out=out)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check_clip(env, ts, norm * 2.0)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check_clip(env, ts, norm * 0.3)


def test_clip_shapes_unaligned_and_extreme_values(env):
    torch, ops = env
    flat = torch.randn(100003, device="cuda")
    check_clip(env, [flat[1:60000], flat[60001:60004], torch.randn(5, 6, 7, device="cuda"), torch.randn((), device="cuda")], 1.0)
    check_clip(env, [torch.full((1000,), 1e30, device="cuda"), torch.full((3,), 1e-40, device="cuda")], 1.0)   # squares overflow 32 bits
    check_clip(env, [torch.full((1000,), 1e-30, device="cuda")], 1e-31)                                        # and vanish in 32 bits
    zeros = [torch.zeros(10, device="cuda")]
    assert float(ops.clip_global_norm(zeros, 1.0)) == 0.0 and (zeros[0] == 0).all()
    for bad in (math.inf, -math.inf, float("nan")):
        t = [torch.randn(5000, device="cuda"), torch.randn(10, device="cuda").to(torch.bfloat16)]
        t[0][777] = bad
        keep = [a.clone() for a in t]
        norm = float(ops.clip_global_norm(t, 0.5))
        assert not math.isfinite(norm)
        assert torch.equal(t[0].view(torch.int32), keep[0].view(torch.int32)) and torch.equal(t[1], keep[1])


# ---------------------------------------------------------------- together ---

def training_step(torch, ops, users, items, bias, ids, targets, weights):
    """One step as a training loop makes it: look up, loss with gradient, lookup's gradient, clip."""
    hidden = ops.embedding_lookup(users, ids, scale=1.25)
    loss, lse, d_hidden, d_items, d_bias = ops.softmax_loss_grad(hidden, items, targets, bias=bias, weights=weights)
    d_users = ops.embedding_lookup_grad(d_hidden, ids, users.shape[0], scale=1.25)
    grads = [d_users, d_items, d_bias]
    norm = ops.clip_global_norm(grads, 0.05)
    return loss, norm, grads


def step_inputs(torch, seed, n=300):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    users = torch.randn(900, 40, generator=g, device="cuda") * 0.4
    items = torch.randn(1203, 40, generator=g, device="cuda") * 0.4
    bias = torch.randn(1203, generator=g, device="cuda") * 0.2
    ids = torch.randint(0, 900, (n,), generator=g, device="cuda", dtype=torch.int32)
    targets = torch.randint(-1, 1203, (n,), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(n, generator=g, device="cuda") / n
    return users, items, bias, ids, targets, weights


def test_training_step_together(env):
    """Against autograd over 64-bit elementary operations."""
    torch, ops = env
    users, items, bias, ids, targets, weights = step_inputs(torch, 1)
    u, i, b = (t.double().requires_grad_() for t in (users, items, bias))
    s = (u[ids.long()] * 1.25) @ i.t() + b
    has = targets >= 0
    each = torch.logsumexp(s, 1) - s.gather(1, targets.long().clamp(0)[:, None]).squeeze(1)
    total = (each * weights.double() * has).sum()
    total.backward()
    norm = math.sqrt(sum(float(t.grad.square().sum()) for t in (u, i, b)))
    loss, got_norm, grads = training_step(torch, ops, users, items, bias, ids, targets, weights)
    # 300 rows x 1203 scores of size < 10 in 32 bits: a probability is off by < 2^-16 relatively, every sum by < 2^-15 of its mass
    assert abs(float(loss.double().sum()) - float(total.detach())) <= 2.0 ** -16 * float((each * weights.double() * has).abs().sum().detach())
    factor = min(1.0, 0.05 / norm)
    mass = weights.double().sum() * float(items.abs().max()) * 2
    assert abs(float(got_norm) - norm) <= 2.0 ** -14 * norm
    for g, t in zip(grads, (u, i, b)):
        assert float((g.double() - t.grad * factor).abs().max()) <= 2.0 ** -15 * float(mass) * factor * 2
    for a, b in zip(training_step(torch, ops, users, items, bias, ids, targets, weights)[2], grads):
        assert torch.equal(a, b)


def test_captured_step_replays(env):
    """The step in a HIP graph, replayed with new inputs in its tensors and eager work between: the eager results, bit for
    bit.  A second graph of the same calls is captured beside it: neither disturbs the other."""
    torch, ops = env
    held = [list(step_inputs(torch, 2)), list(step_inputs(torch, 3))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for h in held:
            training_step(torch, ops, *h)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(training_step(torch, ops, *h))
        graphs.append(g)
    for turn in range(4):
        fresh = [step_inputs(torch, 10 + 2 * turn + j) for j in range(2)]
        want = [training_step(torch, ops, *f) for f in fresh]
        for h, f in zip(held, fresh):
            for a, b in zip(h, f):
                a.copy_(b)
        for g in (graphs if turn % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        for (loss, norm, grads), (l2, n2, g2) in zip(results, want):
            assert torch.equal(loss, l2) and torch.equal(norm, n2)
            assert all(torch.equal(a, b) for a, b in zip(grads, g2))


FORMS = [  # what has a form of its own: few rows, one tile of rows, parts to join or none, short and long lists of ids
    ("loss", 1, 5000, 64, "f32"), ("loss", 2, 3001, 50, "f32"), ("loss", 4, 3001, 51, "f32"), ("loss", 7, 900, 300, "f32"), ("loss", 700, 5000, 64, "f32"),
    ("grad", 3, 9000, 98, "bf16"), ("grad", 60, 20011, 40, "f16"), ("grad", 1003, 50021, 100, "f16"), ("grad", 500, 400, 20, "f32"),
    ("grad", 40, 600, 520, "f32"), ("grad", 0, 50, 8, "f32"),
    ("ids", 300, 1000, 30, "f32"), ("ids", 5000, 90000, 64, "bf16"), ("ids", 80001, 40, 12, "f32"), ("ids", 210001, 300007, 8, "f16"),
    ("bags", 0, 10, 5, "f32"), ("bags", 800, 3000, 33, "f32")]


@pytest.mark.parametrize("kind, rows, vocab, d, dtype", FORMS)
def test_captured_forms_replay(env, kind, rows, vocab, d, dtype):
    torch, ops = env

    def inputs(seed):
        if kind in ("loss", "grad"):
            return make(torch, rows, vocab, d, dtype, seed=seed)
        ids, indptr, values = bags(torch, rows, vocab, 4 if kind == "bags" else 0, seed=seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        if kind == "bags":  # (as many ids for every seed, so that they can be copied)
            indptr = torch.arange(0, 4 * rows + 1, 4, device="cuda", dtype=ids.dtype)
            ids = torch.randint(-1, vocab, (4 * rows,), generator=g, device="cuda").to(ids.dtype)
            values = torch.rand(4 * rows, generator=g, device="cuda")
        x = torch.randn(rows, d, generator=g, device="cuda").to(getattr(torch, DTYPE[dtype]))
        w = torch.randn(vocab, d, generator=g, device="cuda").to(getattr(torch, DTYPE[dtype]))
        return [t for t in (x, w, ids, indptr, values) if t is not None]

    def call(a):
        if kind in ("loss", "grad"):
            return (ops.softmax_loss_grad if kind == "grad" else ops.softmax_loss)(a[0], a[1], a[2], bias=a[3], weights=a[4])
        more = dict(indptr=a[3], values=a[4]) if kind == "bags" else {}
        return ops.embedding_lookup(a[1], a[2], **more), ops.embedding_lookup_grad(a[0], a[2], vocab, **more)

    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = call(held)
    for turn in range(1, 4):
        fresh = inputs(turn)
        want = call(fresh)
        for a, b in zip(held, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for got, exact in zip(results, want):
            assert torch.equal(got, exact)


def test_two_streams_at_once(env):
    torch, ops = env
    sets = [step_inputs(torch, 20 + i, n=900) for i in range(2)]
    want = [training_step(torch, ops, *s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(training_step(torch, ops, *sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for loss, norm, grads in got[i]:
            assert torch.equal(loss, want[i][0]) and torch.equal(norm, want[i][1])
            assert all(torch.equal(a, b) for a, b in zip(grads, want[i][2]))


def test_after_a_session_in_the_same_process(env):
    """LightFM's own library (its own HIP runtime where torch came later) and the operators side by side."""
    torch, ops = env
    import numpy as np
    from lightfm_amd import LightFM
    from tests import helpers as H
    coo = H.make_interactions(60, 50, 700, seed=3)
    m = LightFM(no_components=16, loss="warp", random_state=1).fit(coo, epochs=2)
    w = torch.from_numpy(m.item_embeddings).cuda()
    b = torch.from_numpy(m.item_biases).cuda()
    h = torch.from_numpy(m.user_embeddings).cuda()
    t = torch.arange(60, device="cuda") % 50
    check_softmax(env, h, w, t, b, None)
    assert np.isfinite(m.predict(np.zeros(50, np.int32), np.arange(50, dtype=np.int32))).all()


@pytest.mark.parametrize("max_norm", [0.0, 0.7])
def test_softmax_epochs_are_these_operators(env, max_norm):
    """An epoch of LightFM(loss="softmax") over feature matrices against the same steps made of the operators on torch
    tensors, batch by batch."""
    torch, ops = env
    import numpy as np
    import scipy.sparse as sp
    from lightfm_amd import LightFM
    from lightfm_amd.options import options
    rs = np.random.RandomState(8)
    n_users, n_items, n, d, batch, lr = 90, 130, 1000, 24, 300, 0.05
    coo = sp.coo_matrix((np.ones(n, np.float32), (rs.randint(0, n_users, n), rs.randint(0, n_items, n))), shape=(n_users, n_items))
    fu = sp.random(n_users, 40, 0.1, format="csr", dtype=np.float32, random_state=rs)
    fi = sp.random(n_items, 30, 0.1, format="csr", dtype=np.float32, random_state=rs)
    before = {k: getattr(options, k) for k in ("softmax_batch", "softmax_max_norm", "device_shuffle")}
    m = LightFM(no_components=d, loss="softmax", learning_rate=lr, random_state=4)
    m._initialize(d, 30, 40)
    tables = [torch.from_numpy(getattr(m, name).copy()).cuda() for name in ("user_embeddings", "item_embeddings")]
    bias = torch.zeros(30, 1, device="cuda")
    order = np.arange(n, dtype=np.int32)
    state = np.random.RandomState()
    state.set_state(m.random_state.get_state())
    state.shuffle(order)
    try:
        options.set(softmax_batch=batch, softmax_max_norm=max_norm, device_shuffle=False)
        m.fit_partial(coo, user_features=fu, item_features=fi, epochs=1)
    finally:
        options.set(**before)
    csr = [[torch.from_numpy(v).cuda() for v in (f.indices.astype(np.int32), f.indptr.astype(np.int32), f.data)] for f in (fu, fi)]
    u = torch.from_numpy(coo.row.astype(np.int32)).cuda()
    t = torch.from_numpy(coo.col.astype(np.int32)).cuda()
    weights = tables + [bias]
    accumulators = [torch.ones_like(x) for x in weights]
    for lo in range(0, n, batch):
        pos = torch.from_numpy(order[lo:lo + batch]).cuda().long()
        user, item = (ops.embedding_lookup(tables[s], csr[s][0], indptr=csr[s][1], values=csr[s][2]) for s in (0, 1))
        b = ops.embedding_lookup(bias, csr[1][0], indptr=csr[1][1], values=csr[1][2]).view(-1)
        h = ops.embedding_lookup(user, u[pos])
        _, _, dh, di, db = ops.softmax_loss_grad(h, item, t[pos], bias=b, weights=torch.ones(len(pos), device="cuda"))
        du = ops.embedding_lookup_grad(dh, u[pos], n_users)
        grads = [ops.embedding_lookup_grad(g, csr[s][0], rows, indptr=csr[s][1], values=csr[s][2])
                 for g, s, rows in ((du, 0, 40), (di, 1, 30), (db.view(-1, 1), 1, 30))]
        if max_norm:
            norm = ops.clip_global_norm(grads, max_norm)
        for x, acc, g in zip(weights, accumulators, grads):
            acc.add_(g * g)
            x.sub_(lr * g / acc.sqrt())
    if max_norm:
        assert abs(float(norm) - m._last_epoch_stats[-1]["grad_norm"]) <= 8 * U32 * float(norm)
    # the same kernels in the same order: what may differ is a rounding in each of the four steps' scaling and update
    for x, name in zip(weights, ("user_embeddings", "item_embeddings", "item_biases")):
        want = torch.from_numpy(getattr(m, name)).cuda().view_as(x)
        assert (x - want).abs().max() <= 4 * 8 * U32 * lr + 4 * U32 * want.abs().max(), name


def test_clip_refuses_overlaps_and_tells_autograd(env):
    torch, ops = env
    a = torch.ones(1000, device="cuda")
    b = torch.ones(1000, device="cuda")
    for wrong in (lambda: ops.clip_global_norm([a, a], 1.0), lambda: ops.clip_global_norm([a, a[100:200]], 1.0),
                  lambda: ops.clip_global_norm([a, b], 1.0, out=[b, a]), lambda: ops.clip_global_norm([a[:900], b], 1.0, out=[a[100:], b]),
                  lambda: ops.clip_global_norm([a, b], 1.0, out=[torch.empty_like(a), a]),
                  lambda: ops.clip_global_norm([a, b], 1.0, out=[torch.ones(1000, device="cuda")] * 2)):
        with pytest.raises(ValueError, match="overlaps"):
            wrong()
    assert (a == 1).all() and (b == 1).all()
    assert abs(float(ops.global_norm([a, a])) - math.sqrt(2000.0)) < 1e-4  # (reading twice is no conflict)
    out = torch.empty(2, 1000, device="cuda")
    ops.clip_global_norm([a, a], 1.0, out=[out[0], out[1]])
    assert torch.equal(out[0], out[1])
    before = a._version
    ops.clip_global_norm([a[:500], a[500:]], 1.0)
    assert a._version > before
    with pytest.raises(ValueError, match="negated"):
        ops.global_norm([torch.ones(4, dtype=torch.complex64, device="cuda")[:1].conj().imag])


def test_python_refusals_on_the_gpu(env):
    torch, ops = env
    x, w, t, b, k = make(torch, 6, 20, 8, "f32")
    for wrong in (lambda: ops.softmax_loss(x, w.half(), t), lambda: ops.softmax_loss(x, w[:, :7], t),
                  lambda: ops.softmax_loss(x, w, t[:5]), lambda: ops.softmax_loss(x, w, t.float()),
                  lambda: ops.softmax_loss(x, w, t, bias=b[:3]), lambda: ops.softmax_loss(x, w, t, bias=b.half()),
                  lambda: ops.softmax_loss(x, w, t, weights=k.double()), lambda: ops.softmax_loss(x, w[:0], t),
                  lambda: ops.softmax_loss(x.t(), w, t), lambda: ops.softmax_loss(x[:, :0], w[:, :0], t),
                  lambda: ops.softmax_loss(x, w.cpu(), t), lambda: ops.softmax_loss(x, w.expand(2, 20, 8)[0].t(), t),
                  lambda: ops.softmax_loss(x, w[:1].expand(20, 8), t),
                  lambda: ops.embedding_lookup(w, t.float()), lambda: ops.embedding_lookup(w, t, values=k),
                  lambda: ops.embedding_lookup(w, t, indptr=t[:3].int()),
                  lambda: ops.embedding_lookup_grad(x, t[:4], 20), lambda: ops.embedding_lookup_grad(x, t, 0),
                  lambda: ops.clip_global_norm([x], float("nan")), lambda: ops.clip_global_norm([x, w], 1.0, out=[x]),
                  lambda: ops.clip_global_norm([x.t()], 1.0), lambda: ops.clip_global_norm([x], 1.0, out=[w])):
        with pytest.raises(ValueError):
            wrong()
    with pytest.raises(NotImplementedError):
        ops.softmax_loss(torch.zeros(2, 1025, device="cuda"), torch.zeros(3, 1025, device="cuda"), t[:2])
