"""AdaptedGaussianProjection on the GPU: what it serves and the gradients it trains with, against 64 bits."""
import pickle

import numpy as np
import pytest
import scipy.sparse as sp
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -23


def make(compute, bits=32, **kw):
    from randomprojection_amd import AdaptedGaussianProjection

    rng = np.random.default_rng(1)
    X = rng.standard_normal((500, 301)).astype(np.float32)
    ids = rng.integers(-1, 4, 500)  # adapter 4 has no rows
    est = AdaptedGaussianProjection(n_components=90, n_adapters=5, rank=6, alpha=9.0, random_state=3, compute=compute, state_bits=bits,
                                    chunk_rows=kw.pop("chunk_rows", 200), learning_rate=1e-2, **kw).fit(X)
    return est, X, ids, rng


def rounded(a, compute):
    t = torch.as_tensor(np.asarray(a, np.float32))
    return (t.bfloat16() if compute == "bf16" else t).double().numpy()


@pytest.mark.parametrize("compute", ["fp32", "bf16"])
def test_transform(compute):
    est, X, ids, rng = make(compute)
    est._up = rng.standard_normal(est._up.shape).astype(np.float32)  # as after training
    Y = est.transform(X, adapters=ids)
    x, c, d, u = (rounded(a, compute) for a in (X, est.components_, est.down_, est.up_))
    want, size = x @ c.T, abs(x) @ abs(c).T
    for g in range(5):
        at = ids == g
        want[at] += 1.5 * (x[at] @ d[g].T @ u[g])
        size[at] += 1.5 * (abs(x[at]) @ abs(d[g]).T @ abs(u[g]))
    assert Y.dtype == np.float32 and (abs(Y - want) <= (301 + 6 + 8) * E * size).all()
    assert np.array_equal(est.transform(sp.csr_matrix(X), adapters=ids), Y)
    from randomprojection_amd.gaussian import GaussianRandomProjection

    base = GaussianRandomProjection(n_components=90, random_state=3, compute=compute if compute == "bf16" else "auto").fit(X)
    assert np.array_equal(est.transform(X), base.transform(X))


@pytest.mark.parametrize("compute", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_partial_fit(bits, compute):
    """The first step's first moments are a tenth of the gradient; adapters without rows keep everything; two estimators of one history are
    the same bit for bit, also through a pickle."""
    est, X, ids, rng = make(compute, bits, chunk_rows=1000)
    est._up = (rng.standard_normal(est._up.shape) * 0.1).astype(np.float32)
    other = pickle.loads(pickle.dumps(est))
    T = rng.standard_normal((500, 90)).astype(np.float32)
    before = est.down_.copy(), est.up_.copy()
    est.partial_fit(X, T, ids)
    x, c, d, u = (rounded(a, compute) for a in (X, est.components_, *before))
    y = x @ c.T
    for g in range(4):
        y[ids == g] += 1.5 * (x[ids == g] @ d[g].T @ u[g])
    # the distance is taken of y in f32 and rounded to the compute type: half a step, and what y is off by (K steps of at most |y|'s parts)
    dy = (y - T) * 2 / 500
    slack = np.abs(dy) * (2.0 ** -8 if compute == "bf16" else 2.0 ** -22) + 330 * E * (abs(x) @ abs(c).T + 60) * 2 / 500
    assert est.loss_ == pytest.approx(((y - T) ** 2).sum(1).mean(), rel=1e-4)
    held = est._bank.opt.state_values()[0].cpu().double().numpy() / 0.1
    mk, pk = est._bank.params[0].shape[-1], est._bank.params[1].shape[-1]
    each = [-(-6 * k // 256) * 256 for k in [mk] * 5 + [pk] * 5]
    at = np.concatenate([[0], np.cumsum(each)])
    for g in range(5):
        rows = ids == g
        dd = 1.5 * (dy[rows] @ u[g].T).T @ x[rows]
        du = 1.5 * (x[rows] @ d[g].T).T @ dy[rows]
        ed = 1.5 * (slack[rows] @ abs(u[g]).T).T @ abs(x[rows]) + (500 + 90) * E * 1.5 * (abs(dy[rows]) @ abs(u[g]).T).T @ abs(x[rows])
        eu = 1.5 * (abs(x[rows]) @ abs(d[g]).T).T @ (slack[rows] + (500 + 301) * E * abs(dy[rows]))
        for want, err, start, width, k in ((dd, ed, at[g], mk, 301), (du, eu, at[5 + g], pk, 90)):
            got = held[start:start + 6 * width].reshape(6, width)
            assert not got[:, k:].any()
            # 8 bits: at most one code, an eighth of the value or of the least binade (2^-14 of the block's largest)
            coarse = 0.126 * abs(want) + 2.0 ** -14 * np.abs(want).max() if bits == 8 and rows.any() else 1e-6 * abs(want)
            assert (abs(got[:, :k] - want) <= err * 1.01 + coarse + 1e-30).all(), (g, k)
    assert np.array_equal(est.down_[4], before[0][4]) and np.array_equal(est.up_[4], before[1][4])
    assert not np.array_equal(est.down_[3], before[0][3])
    for _ in range(2):
        est.partial_fit(X, T, ids)
    other.partial_fit(X, T, ids)
    other = pickle.loads(pickle.dumps(other))
    for _ in range(2):
        other.partial_fit(X, T, ids)
    assert np.array_equal(est.down_, other.down_) and np.array_equal(est.up_, other.up_)
    assert np.array_equal(est.transform(X, adapters=ids), other.transform(X, adapters=ids))


def test_parameters_set_after_fit():
    """They hold from the next call on; what the states' layout depends on is refused once a step was taken."""
    est, X, ids, rng = make("fp32")
    T = rng.standard_normal((500, 90)).astype(np.float32)
    bf = pickle.loads(pickle.dumps(est))
    first = bf.transform(X, adapters=ids)
    bf.set_params(compute="bf16")  # no step yet
    assert not np.array_equal(bf.transform(X, adapters=ids), first) and bf._bank.low[0].dtype == torch.bfloat16
    est.partial_fit(X, T, ids)
    down, up = est.down_, est.up_
    est.set_params(learning_rate=0.0, alpha=0.0, n_adapters=9, rank=2).partial_fit(X, T, ids)
    assert np.array_equal(est.down_, down) and np.array_equal(est.up_, up)
    shared = est.transform(X, adapters=np.full(500, -1))
    assert np.array_equal(est.transform(X, adapters=ids), shared)
    est.set_params(alpha=9.0)
    assert not np.array_equal(est.transform(X, adapters=ids)[ids >= 0], shared[ids >= 0])
    with pytest.raises(ValueError, match="-1 .. 4"):
        est.transform(X, adapters=np.full(500, 5))
    for change, back in (({"compute": "bf16"}, {"compute": "fp32"}), ({"state_bits": 8}, {"state_bits": 32})):
        with pytest.raises(ValueError, match="cannot change"):
            est.set_params(**change).transform(X, adapters=ids)
        est.set_params(**back)
    assert np.array_equal(est.down_, down)
    with pytest.raises(ValueError, match="NaN"):
        est.partial_fit(X, np.full_like(T, np.nan), ids)
