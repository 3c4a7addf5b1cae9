"""LightFM(loss="softmax"): epochs of the whole-catalogue cross entropy (include/lfm_hip.h: lfm_session_epoch_softmax),
which run the embedding lookup, the softmax loss with its gradients, the sorted lookup gradients and the clipping norm
one after the other.  The reference has no such loss; the oracle is the formula in float64."""
import os
import pickle
import re
import subprocess
import sys

import numpy as np
import pytest
import scipy.sparse as sp

from lightfm_amd import LightFM, _native
from lightfm_amd.options import options

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def restore_options():
    before = {k: getattr(options, k) for k in ("softmax_batch", "softmax_max_norm", "device_shuffle", "mode")}
    yield
    options.set(**before)


# ------------------------------------------------------------------ without a device

def test_struct_layout_matches_the_header(tmp_path):
    fields = [f for f, _ in _native.LfmSoftmaxEpoch._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "lfm_hip.h"\nint main(void){printf("%%zu", sizeof(lfm_softmax_epoch));\n%s\nreturn 0;}\n'
                   % "\n".join('printf(" %%zu", offsetof(lfm_softmax_epoch, %s));' % f for f in fields))
    exe = str(tmp_path / "probe")
    subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = [int(v) for v in subprocess.check_output([exe]).split()]
    assert got[0] == _native.C.sizeof(_native.LfmSoftmaxEpoch)
    assert got[1:] == [getattr(_native.LfmSoftmaxEpoch, f).offset for f in fields]
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "lfm_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct lfm_softmax_epoch \{(.*?)\} lfm_softmax_epoch;", header, flags=re.S).group(1)
    assert sum(len(stmt.split(",")) for stmt in body.split(";") if stmt.strip()) == len(fields)


def test_estimator_interface():
    m = LightFM(loss="softmax", no_components=4)
    assert m.get_params()["loss"] == "softmax"
    assert LightFM().set_params(loss="softmax").loss == "softmax"
    with pytest.raises(AssertionError):
        LightFM(loss="softmax-ce")
    with pytest.raises(ValueError):
        options.set(softmax_batches=3)


def test_refusals_without_a_device():
    from lightfm_amd.distributed import DistributedFit
    lib = _native.lib()
    assert lib.lfm_session_epoch_softmax(None, 0, _native.C.c_double(0), _native.C.c_double(0), None) == -1
    with pytest.raises(NotImplementedError, match="one device"):
        DistributedFit(LightFM(loss="softmax"), sp.coo_matrix(np.eye(4, dtype=np.float32)), 0, 1, None)
    if _native.device_count() == 0:
        with pytest.raises(_native.HipBackendError):
            LightFM(loss="softmax").fit(sp.coo_matrix(np.eye(4, dtype=np.float32)))


# ------------------------------------------------------------------ against the formula

class Oracle(object):
    """One table: weights and accumulators in float64, stepped with a batch's summed gradient."""

    def __init__(self, W, G, M, model):
        self.W, self.G, self.M = (a.astype(np.float64).copy() for a in (W, G, M))
        self.model, self.slack = model, 0.0

    def step(self, g, mass, l2):
        """mass: the sum of the magnitudes of what g adds up -- what a relative error of its terms multiplies."""
        g = g + l2 * self.W
        on = g != 0
        m = self.model
        if m.learning_schedule == "adadelta":
            acc = m.rho * self.G + (1 - m.rho) * g * g
            rate = np.sqrt(self.M + m.epsilon) / np.sqrt(acc + m.epsilon)
            mom = m.rho * self.M + (1 - m.rho) * (rate * g) ** 2
            self.M = np.where(on, mom, self.M)
        else:
            acc = self.G + g * g
            rate = m.learning_rate / np.sqrt(acc)
        self.W = np.where(on, self.W - rate * g, self.W)
        self.G = np.where(on, acc, self.G)
        # d(step)/dg <= the largest rate; the terms of g are good to 2^-19: products and sums in float32 (2^-24 each, a dozen
        # of them one after the other), exp of scores that are good to 2^-22 of |x||w| <= 2, hi/lo halves of 2^-22
        self.slack += float((rate * (mass + np.abs(l2 * self.W))).max()) * 2.0 ** -19

    def check(self, W, G, steps):
        # a step's error moves the later scores and with them the later gradients: twice the sum over the few steps here;
        # and W is rounded once per step
        tol = 2 * self.slack + steps * 2.0 ** -24 * np.abs(self.W).max()
        assert np.abs(W - self.W).max() <= tol, (np.abs(W - self.W).max(), tol)
        # the accumulator: 2 |g| dg + rounding
        assert np.abs(G - self.G).max() <= 2.0 ** -16 * max(1.0, np.abs(self.G).max())


def softmax_epoch_oracle(m, coo, weight, fu, fi, order, batch, max_norm, start):
    FU, FI = fu.toarray().astype(np.float64), fi.toarray().astype(np.float64)
    user = Oracle(*start["user"], m)
    item = Oracle(*start["item"], m)
    bias = Oracle(*start["bias"], m)
    total, targets, norm, steps = 0.0, 0, 0.0, 0
    for lo in range(0, len(order), batch):
        pos = order[lo:lo + batch]
        u, t, w = coo.row[pos], coo.col[pos], weight[pos].astype(np.float64)
        on = coo.data[pos] > 0
        X, V, b = FU @ user.W, FI @ item.W, FI @ bias.W
        S = X[u] @ V.T + b
        top = S.max(axis=1, keepdims=True)
        lse = (top + np.log(np.exp(S - top).sum(axis=1, keepdims=True)))[:, 0]
        rows = np.arange(len(pos))
        total += float((w * (lse - S[rows, t]))[on].sum())
        targets += int(on.sum())
        q = np.exp(S - lse[:, None])
        q[rows, t] -= 1.0
        q *= (w * on)[:, None]
        dX = np.zeros_like(X)
        np.add.at(dX, u, q @ V)
        aX = np.zeros_like(X)
        np.add.at(aX, u, np.abs(q) @ np.abs(V))
        dV, aV = q.T @ X[u], np.abs(q).T @ np.abs(X[u])
        g = [FU.T @ dX, FI.T @ dV, FI.T @ q.sum(axis=0)]
        mass = [np.abs(FU).T @ aX, np.abs(FI).T @ aV, np.abs(FI).T @ np.abs(q).sum(axis=0)]
        norm = float(np.sqrt(sum((x * x).sum() for x in g)))
        scale = min(1.0, max_norm / norm) if max_norm > 0 and norm > 0 else 1.0
        l2 = (m.user_alpha * len(pos), m.item_alpha * len(pos), m.item_alpha * len(pos))
        for table, gg, aa, r in zip((user, item, bias), g, mass, l2):
            table.step(gg * scale, aa * scale, r)
        steps += 1
    return user, item, bias, total / max(1, targets), targets, norm, steps


def make_data(seed, n_users, n_items, n, negatives=False):
    rs = np.random.RandomState(seed)
    coo = sp.coo_matrix((rs.choice([1.0, -1.0, 0.5, 0.0] if negatives else [1.0], size=n).astype(np.float32),
                         (rs.randint(0, n_users, n).astype(np.int32), rs.randint(0, n_items, n).astype(np.int32))),
                        shape=(n_users, n_items))
    return coo, rs


def features(rs, rows, cols):
    """Rows of one to five features with values of either sign; row 1 has none."""
    f = sp.lil_matrix((rows, cols), dtype=np.float32)
    for r in range(rows):
        if r != 1:
            for c in rs.choice(cols, size=rs.randint(1, 6), replace=False):
                f[r, c] = rs.uniform(-1, 1.5)
    return f.tocsr()


CASES = [
    # users, items, interactions, d, batch, model arguments, max_norm, features, negatives, weights
    (40, 30, 200, 10, 64, {}, 0.0, "", False, False),
    (40, 30, 200, 10, 64, {}, 2.0, "", False, False),
    (1, 1, 3, 1, 1, {}, 0.0, "", False, False),
    (7, 2, 9, 3, 4, {}, 0.0, "", False, True),
    (300, 515, 1100, 33, 512, {}, 0.0, "", True, True),
    (40, 30, 200, 16, 100, dict(learning_schedule="adadelta"), 0.0, "", False, False),
    (60, 50, 333, 20, 128, dict(item_alpha=1e-3, user_alpha=2e-3), 1.5, "", True, True),
    (50, 64, 400, 12, 150, {}, 0.0, "ui", False, True),
    (50, 64, 400, 64, 150, {}, 3.0, "i", True, False),
    (50, 64, 400, 65, 400, dict(learning_schedule="adadelta", item_alpha=1e-4), 0.0, "u", False, False),
    (20, 40, 90, 300, 32, {}, 0.0, "ui", False, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%du_%di_%d_d%d_%s" % (c[0], c[1], c[2], c[3], c[7]))
def test_epoch_against_the_formula(case):
    n_users, n_items, n, d, batch, kw, max_norm, feats, negatives, weights = case
    coo, rs = make_data(n + d, n_users, n_items, n, negatives)
    # one more row of features than users: representations of items / users nobody interacts with
    fu = features(rs, n_users + 1, 23) if "u" in feats else sp.identity(n_users, dtype=np.float32, format="csr")
    fi = features(rs, n_items, 19) if "i" in feats else sp.identity(n_items, dtype=np.float32, format="csr")
    weight = rs.uniform(0.5, 2.0, n).astype(np.float32) if weights else np.ones(n, np.float32)
    options.set(softmax_batch=batch, softmax_max_norm=max_norm, device_shuffle=False)
    m = LightFM(no_components=d, loss="softmax", learning_rate=0.1, random_state=5, **kw)
    m._initialize(d, fi.shape[1], fu.shape[1])
    scale = np.float32(d ** 0.5)  # representations of unit size, so that the scores are not all alike
    m.item_embeddings *= scale
    m.user_embeddings *= scale
    m.item_biases += rs.uniform(-1, 1, fi.shape[1]).astype(np.float32)
    m.user_biases += rs.uniform(-1, 1, fu.shape[1]).astype(np.float32)
    user_biases = m.user_biases.copy()
    start = {"user": (m.user_embeddings.copy(), m.user_embedding_gradients.copy(), m.user_embedding_momentum.copy()),
             "item": (m.item_embeddings.copy(), m.item_embedding_gradients.copy(), m.item_embedding_momentum.copy()),
             "bias": (m.item_biases.copy(), m.item_bias_gradients.copy(), m.item_bias_momentum.copy())}
    order = np.arange(n, dtype=np.int32)
    state = np.random.RandomState()
    state.set_state(m.random_state.get_state())
    state.shuffle(order)
    sample_weight = sp.coo_matrix((weight, (coo.row, coo.col)), shape=coo.shape) if weights else None
    m.fit_partial(coo, user_features=fu if "u" in feats else None, item_features=fi if "i" in feats else None,
                  sample_weight=sample_weight, epochs=1)
    user, item, bias, loss, targets, norm, steps = softmax_epoch_oracle(m, coo, weight, fu, fi, order, batch, max_norm, start)
    stats = m._last_epoch_stats[-1]
    assert (stats["steps"], stats["targets"]) == (steps, targets)
    assert abs(stats["loss"] - loss) <= 2.0 ** -16 * max(1.0, abs(loss))
    if max_norm > 0:
        assert abs(stats["grad_norm"] - norm) <= 2.0 ** -14 * norm
    user.check(m.user_embeddings, m.user_embedding_gradients, steps)
    item.check(m.item_embeddings, m.item_embedding_gradients, steps)
    bias.check(m.item_biases, m.item_bias_gradients, steps)
    assert np.array_equal(m.user_biases, user_biases)


@pytest.mark.gpu
def test_the_same_bits_every_time():
    coo, _ = make_data(1, 500, 300, 6000)
    fitted = []
    for mode in ("parallel", "serial", "parallel"):
        options.set(mode=mode, softmax_batch=512, softmax_max_norm=5.0)
        m = LightFM(no_components=24, loss="softmax", random_state=np.random.RandomState(3)).fit(coo, epochs=3)
        fitted.append(m)
        assert [s["targets"] for s in m._last_epoch_stats] == [6000] * 3
    for m in fitted[1:]:
        for name in ("item_embeddings", "item_embedding_gradients", "item_biases", "user_embeddings"):
            assert np.array_equal(getattr(m, name), getattr(fitted[0], name)), name
    again = pickle.loads(pickle.dumps(fitted[0]))
    ids = np.arange(300, dtype=np.int32)
    assert np.array_equal(again.predict(7, ids), fitted[0].predict(7, ids))


@pytest.mark.gpu
def test_epochs_without_targets_leave_the_model():
    coo, _ = make_data(2, 30, 20, 50)
    coo.data[:] = -1.0
    m = LightFM(no_components=8, loss="softmax", random_state=1)
    m._initialize(8, 20, 30)
    before = m.item_embeddings.copy(), m.user_embeddings.copy()
    m.fit_partial(coo, epochs=2)
    assert m._last_epoch_stats[-1]["targets"] == 0 and m._last_epoch_stats[-1]["loss"] == 0.0
    assert np.array_equal(before[0], m.item_embeddings) and np.array_equal(before[1], m.user_embeddings)
    empty = sp.coo_matrix((30, 20), dtype=np.float32)
    m.fit_partial(empty, epochs=1)
    assert m._last_epoch_stats[-1]["steps"] == 0
    assert np.array_equal(before[0], m.item_embeddings)


@pytest.mark.gpu
def test_operators_after_a_fit():
    """A process that has trained before it imports torch can still use torch and the operators on the GPU."""
    script = """
import numpy as np, scipy.sparse as sp
from lightfm_amd import LightFM
coo = sp.coo_matrix(np.ones((20, 30), np.float32))
m = LightFM(no_components=8, loss="softmax", random_state=1).fit(coo)
import torch
from lightfm_amd import operators
w = torch.from_numpy(m.item_embeddings).cuda()
loss, lse = operators.softmax_loss(w, w, torch.arange(30, device="cuda"))
want = torch.nn.functional.cross_entropy(w.cpu().double() @ w.cpu().double().t(), torch.arange(30), reduction="none")
assert (loss.cpu().double() - want).abs().max() < 1e-5
m.fit(coo)
print("finished")
"""
    out = subprocess.run([sys.executable, "-u", "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert out.returncode == 0 and "finished" in out.stdout, out.stderr[-2000:]


@pytest.mark.gpu
def test_feature_matrices_without_entries():
    """Every representation is zero: a uniform softmax, log(items) per target, and nothing to learn from."""
    coo, _ = make_data(4, 30, 20, 64)
    m = LightFM(no_components=8, loss="softmax", random_state=1)
    m._initialize(8, 5, 6)
    before = m.item_embeddings.copy(), m.user_embeddings.copy()
    m.fit_partial(coo, user_features=sp.csr_matrix((30, 6), dtype=np.float32), item_features=sp.csr_matrix((20, 5), dtype=np.float32))
    assert abs(m._last_epoch_stats[-1]["loss"] - np.log(20)) <= 2.0 ** -20 * np.log(20)
    assert np.array_equal(before[0], m.item_embeddings) and np.array_equal(before[1], m.user_embeddings)
    assert not m.item_biases.any()


@pytest.mark.gpu
def test_refused_options_and_divergence():
    coo, _ = make_data(3, 30, 20, 50)
    m = LightFM(no_components=8, loss="softmax", random_state=1)
    for bad in (dict(softmax_batch=-1), dict(softmax_batch=(1 << 32) + 5), dict(softmax_max_norm=-1.0), dict(softmax_max_norm=float("nan"))):
        options.set(softmax_batch=0, softmax_max_norm=0.0)
        options.set(**bad)
        with pytest.raises(ValueError):
            m.fit_partial(coo)
    options.set(softmax_batch=0, softmax_max_norm=0.0)
    with pytest.raises(ValueError, match="not.*finite|finite"):
        LightFM(no_components=8, loss="softmax", learning_rate=1e38, random_state=1).fit(coo, epochs=10)
