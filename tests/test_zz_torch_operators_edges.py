"""The softmax operators where a row, an item or a whole batch is out of the ordinary: values that are not finite, targets
that are masked, rows without a target that are far larger than the others, batches without any target, probabilities far
below the others.  Bounds are derived as in test_zz_torch_operators."""
import math

import pytest

from tests.test_zz_torch_operators import U32, env, make, near, reference  # noqa: F401  (env is a fixture)

pytestmark = pytest.mark.gpu

FORMS = [(1, 64), (3, 40), (4, 51), (7, 300), (90, 64), (90, 50), (70, 300), (2500, 64)]


def both(ops, x, w, t, b, k):
    """The loss alone and with its gradients (forms of their own where there are few rows)."""
    return ops.softmax_loss(x, w, t, bias=b, weights=k), ops.softmax_loss_grad(x, w, t, bias=b, weights=k)


# ---------------------------------------------------------------- not finite ---

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, d", FORMS)
def test_lse_of_rows_that_are_not_numbers(env, rows, d, dtype):
    """A hidden row of NaN has a lse of NaN, with a target (and then its loss is NaN) and without one (loss 0).  The other
    rows have the bits that they have beside rows of zeros."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 333, d, dtype, seed=31, ignored=False)
    lost = torch.zeros(rows, dtype=torch.bool, device="cuda")
    lost[[0, rows // 2, rows - 1]] = True
    t[rows - 1] = -1
    clean = both(ops, torch.where(lost[:, None], torch.zeros_like(x), x), w, t, b, k)
    x[lost] = float("nan")
    for got, want in zip(both(ops, x, w, t, b, k), clean):
        assert torch.isnan(got[1][lost]).all()
        assert torch.equal(got[1][~lost], want[1][~lost]) and torch.equal(got[0][~lost], want[0][~lost])
        assert (got[0][t < 0] == 0).all() and torch.isnan(got[0][lost & (t >= 0)]).all()


# ------------------------------------------------------------ masked targets ---

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, d", FORMS)
@pytest.mark.parametrize("left", [True, False])
def test_targets_that_are_removed_items(env, rows, d, dtype, left):
    """A target whose bias is -inf and whose row holds NaN or infinities: its loss is infinite, everything else is what it is
    with a row of zeros, bit for bit.  left: there are items besides the removed ones."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 333, d, dtype, seed=32, ignored=False)
    b[[5, 64, 200, 332]] = -math.inf
    if not left:
        b[:] = -math.inf
    w[[5, 64, 200, 332]] = 0
    t[0], t[rows // 2], t[rows - 1] = 5, 64, 332
    if rows > 10:
        t[3] = 200
    out = torch.isinf(b[t.long()])
    clean = both(ops, x, w, t, b, k)
    w[5], w[64], w[200] = float("nan"), math.inf, -math.inf
    w[332, d // 2] = float("nan")
    for got, want in zip(both(ops, x, w, t, b, k), clean):
        assert (got[0][out] == math.inf).all() and torch.isfinite(got[0][~out]).all()
        for i, (g, c) in enumerate(zip(got, want)):
            assert torch.equal(g, c), i
            if i > 1:
                assert torch.isfinite(g).all(), i


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", [-1e30, -3.402823466e38])
@pytest.mark.parametrize("rows, d", [(1, 64), (3, 40), (7, 300), (90, 64), (70, 300), (2500, 64)])
def test_targets_that_are_masked_items(env, rows, d, dtype, mask):
    """A target whose bias is a large negative number, as masks are: loss = weight (lse - score).  The score is the mask
    to within half a step of float32, lse is of the order of 10: two roundings, and one of the product with the weight.  The
    gradients are those with -inf for a mask, but for what the scores' own rounding does to the others: nothing."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 333, d, dtype, seed=33, ignored=False, size=0.05)
    k = k * 0.5
    t[t < 20] = 77
    b[5:15] = mask
    w[5:15] *= 0.5  # (no row's size rests on them)
    t[0], t[rows // 2] = 7, 9
    out = b[t.long()] < -1e20
    inf = torch.where(b < -1e20, torch.full_like(b, -math.inf), b)
    for got, want in zip(both(ops, x, w, t, b, k), both(ops, x, w, t, inf, k)):
        exact = k.double() * -b[t.long()].double()
        assert ((got[0].double() - exact).abs() <= 4 * U32 * exact)[out].all(), (got[0][out][:4].tolist(), exact[out][:4].tolist())
        assert torch.equal(got[0][~out], want[0][~out])
        for i in range(1, len(got)):
            assert torch.equal(got[i], want[i]), i


# -------------------------------------------------------- rows without target ---

def lse_bound(torch, x, w, b):
    """(lse, bound) in 64 bits, a piece of the rows at a time."""
    values, bounds = [], []
    for lo in range(0, x.shape[0], 256):
        t = torch.zeros(min(256, x.shape[0] - lo), dtype=torch.int64, device="cuda")
        value, bound = reference(torch, x[lo:lo + 256], w, t, b, None)
        values.append(value[1])
        bounds.append(bound[1])
    return torch.cat(values), torch.cat(bounds)


@pytest.mark.parametrize("base, size", [(1.0, 20.0), (1.0, 1e4), (1.0, 1e30), (1e-18, 1e18), (1e-18, 1e12)])
@pytest.mark.parametrize("rows, vocab, d", [(40, 2003, 64), (90, 333, 50), (40, 500, 300), (2500, 700, 64)])
def test_large_rows_without_target(env, rows, vocab, d, base, size):
    """Finite rows without a target, far larger than the rows with one: their lse is right, the others keep their bits."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, vocab, d, "f32", seed=34, ignored=False)
    x *= base
    b[vocab // 2] = -math.inf
    t[t == vocab // 2] = 1
    out = torch.zeros(rows, dtype=torch.bool, device="cuda")
    out[::3] = True
    out[rows - 1] = True
    t[out] = -1
    clean = both(ops, torch.where(out[:, None], torch.zeros_like(x), x), w, t, b, k)
    x = torch.where(out[:, None], x * size, x)
    x[3] = x[3] * 0 + 2.0 ** -100
    x[6] = 0.0
    x[9, d - 1] = float("nan")
    lost = torch.isnan(x).any(1)
    value, bound = lse_bound(torch, torch.where(lost[:, None], torch.zeros_like(x), x), w, b)
    for got, want in zip(both(ops, x, w, t, b, k), clean):
        for i in range(len(got)):
            if i != 1:
                assert torch.equal(got[i], want[i]), i
        assert torch.equal(got[1][~out], want[1][~out])
        assert torch.isnan(got[1][lost]).all()
        near(torch, got[1][~lost], value[~lost], bound[~lost], "lse")


@pytest.mark.parametrize("d", [64, 300])
def test_large_rows_without_target_cost_no_more_than_others(env, d):
    """A padded batch whose padding holds large values takes the time of one whose padding is zero (a third of the rows here;
    scored apart from the sweep they cost tens of times the batch)."""
    torch, ops = env
    x, w, t, b, k = make(torch, 4096, 20011, d, "f32", seed=35, ignored=False)
    out = torch.arange(4096, device="cuda") % 3 == 0
    t[out] = -1
    zero, large = torch.where(out[:, None], torch.zeros_like(x), x), torch.where(out[:, None], x * 1e3, x)

    def best(x):
        ops.softmax_loss(x, w, t, bias=b, weights=k)
        times = []
        for _ in range(5):
            one, two = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            one.record()
            ops.softmax_loss(x, w, t, bias=b, weights=k)
            two.record()
            torch.cuda.synchronize()
            times.append(one.elapsed_time(two))
        return min(times)

    assert best(large) <= 2.0 * best(zero)


@pytest.mark.parametrize("rows, vocab, d", [(3, 333, 40), (7, 900, 50), (90, 333, 64), (2500, 400, 40), (60, 300, 300)])
def test_batches_without_any_target(env, rows, vocab, d):
    """Tiny rows against a large table with nothing to train on: lse keeps its precision."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, vocab, d, "f32", seed=36)
    x, w = x * 1e-6, w * 1e6
    t[:] = -1
    value, bound = lse_bound(torch, x, w, b)
    for got in both(ops, x, w, t, b, k):
        assert (got[0] == 0).all()
        near(torch, got[1], value, bound, "lse")
        assert all((g == 0).all() for g in got[2:])


# ------------------------------------------------------------------- precision ---

@pytest.mark.parametrize("vocab", [20011, 200003])
def test_float32_terms_keep_their_bits_in_a_large_vocabulary(env, vocab):
    """All items but 40 have a bias of -40: their terms, below 2^-45 of the row's largest, vanish in the split halves, so that
    however large the table is a sum has 40 terms and its bound is as small.  (m a multiple of ln 2 apart: at most 40
    rescalings.)  d_hidden: a probability is off by its score, twice (own and lse's), its own split 2^-21, the 40 + 40
    roundings of sum and rescalings.  The tail itself is vocab exp(-40) exp(2 max |s|) of the sum.  Probabilities rounded to one float16 half
    are outside the bound: asserted as well."""
    torch, ops = env
    rows, d = 40, 64
    x, w, t, b, k = make(torch, rows, vocab, d, "f32", seed=37, ignored=False)
    x, w = (torch.round(a * 64) / 64 for a in (x, w))  # products and their sums are exact: multiples of 2^-12 below 2^11
    live = torch.randperm(vocab, generator=torch.Generator().manual_seed(2))[:40].cuda()
    b[:] = -40.0
    b[live] = 0.25
    t = live[torch.arange(rows, device="cuda") % 40]
    xx, ww, g = x.double(), w.double(), k.double()[:, None]
    s = xx @ ww[live].t() + 0.25
    rest = torch.logsumexp(xx @ ww.t() + b.double(), 1)
    lse = torch.logsumexp(s, 1)
    tail = float((rest - lse).max()) + 2.0 ** -40
    assert tail < 2.0 ** -26
    top = float(s.abs().max())
    p = torch.exp(s - rest[:, None])
    hot = (t[:, None] == live[None, :]).double()
    rel = 2 * 4 * U32 * top + (40 + 64) * U32 + 8 * U32 * (1 + top) + 16 * U32 + tail
    half, sums = 2.0 ** -21, (40 + 40 + 16) * U32
    q = g * (p - hot)
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)
    bx = (rel + half + sums + tail) * g * ((p + hot) @ ww[live].abs())
    near(torch, got[2], q @ ww[live], bx + 2 * U32 * (q @ ww[live]).abs() + 2.0 ** -30, "d_hidden")
    bw = ((rel + half) * g * p + (rel + half + sums) * q.abs() + 2.0 ** -38 * g.max()).t() @ xx.abs()
    near(torch, got[3][live], q.t() @ xx, bw + 2 * U32 * (q.t() @ xx).abs(), "d_table")
    # 2^7 p and 2^14 q / 2^e in one half
    e = math.ceil(math.log2(float(k.max())))
    single = g * ((p * 128).half().double() / 128 - hot) @ ww[live]
    assert ((single - q @ ww[live]).abs() > bx).any()
    single = ((q * 2.0 ** (14 - e)).half().double() * 2.0 ** (e - 14)).t() @ xx
    assert ((single - q.t() @ xx).abs() > bw).any()


@pytest.mark.parametrize("rows", [40, 300])
def test_float32_gradients_of_unlikely_items(env, rows):
    """Items of probabilities about 2^-24 to 2^-37: the terms of d_table keep 22 bits and an absolute error of 2^-38 of the largest
    weight, as lfm_ops.h says."""
    torch, ops = env
    x, w, t, b, k = make(torch, rows, 700, 48, "f32", seed=38, ignored=False)
    rare = torch.arange(200, 600, device="cuda")
    b[rare] = -math.log(2.0) * (12.0 + 13.0 * torch.rand(400, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    t[(t >= 200) & (t < 600)] = 11
    (_, _, _, dw, _), _ = reference(torch, x, w, t, b, k)
    xx, ww = x.double(), w.double()
    s = xx @ ww.t() + b.double()
    q = k.double()[:, None] * torch.exp(s - torch.logsumexp(s, 1)[:, None])
    ds = (48 * U32 + 2.0 ** -20) * (xx.abs() @ ww.abs().t()) + 8 * U32 * s.abs()
    rel = ds + ds.max(1).values[:, None] + (700 + 64 + 40) * U32 + 2.0 ** -21 + 2.0 ** -20 + rows * U32
    bound = (rel * q).t() @ xx.abs() + 2.0 ** -38 * float(k.max()) * xx.abs().sum(0) + 2 * U32 * dw.abs()
    got = ops.softmax_loss_grad(x, w, t, bias=b, weights=k)[3]
    near(torch, got[rare], dw[rare], bound[rare], "d_table")
    # (a floor of 2^-26 of the largest weight would show)
    assert (q[:, rare].t() @ xx.abs() > 4 * bound[rare]).any(1).float().mean() > 0.9


# ------------------------------------------------------------------------ clip ---

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_clip_by_a_factor_below_the_normal_numbers(env, dtype):
    """max_norm / norm < 2^-126: the factor has its bits all the same.  Off by a rounding to float32, one to the result's type
    and the factor's own."""
    torch, ops = env
    x = (torch.randn(70001, device="cuda") * 1e30).to(getattr(torch, dtype))
    norm = math.sqrt(float(x.double().square().sum()))
    for top in (1e-7, 3e-9):
        out = [torch.empty_like(x), torch.empty_like(x[1:])]
        got = ops.clip_global_norm([x, x[1:]], top, out=out)
        both = math.sqrt(norm ** 2 + float(x[1:].double().square().sum()))
        assert abs(float(got) - both) <= 2 * U32 * both
        for o, t in zip(out, (x, x[1:])):
            want = t.double() * (top / both)
            near(torch, o, want, (torch.finfo(x.dtype).eps / 2 + 4 * U32) * want.abs() + 2.0 ** -149, "clipped")


def test_clip_of_a_norm_beyond_float32(env):
    """1e39 from finite values: reported as infinite, the values are scaled by it."""
    torch, ops = env
    x = torch.full((100,), 1e38, device="cuda")
    assert float(ops.clip_global_norm([x], 2.0)) == math.inf
    near(torch, x, torch.full((100,), 0.2, dtype=torch.float64, device="cuda"), torch.tensor(0.2 * 4 * U32, device="cuda").double(), "clipped")
