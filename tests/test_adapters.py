"""Adapters beside the dense projection and AdamW: what is refused, checked without a GPU."""
import ctypes

import pytest
import torch

from randomprojection_amd import _native as nat
from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device, prepare_bank
from randomprojection_amd.optim import AdamW


def _forward_args(n=5, m=70, p=9, G=3, R=2):
    return {"X": torch.randn(n, m), "C": torch.randn(p, m), "down": torch.randn(G, R, m), "up": torch.randn(G, R, p),
            "ids": torch.zeros(n, dtype=torch.int32)}


@pytest.mark.parametrize("change,match", [
    ({"X": torch.randn(70)}, "2-D"),
    ({"C": torch.randn(9, 71)}, "C must have shape"),
    ({"C": torch.randn(9)}, "C must be 2-D"),
    ({"down": torch.randn(3, 2, 71)}, "down must have shape"),
    ({"up": torch.randn(3, 2, 8)}, "up must have shape"),
    ({"up": torch.randn(3, 1, 9)}, "same, positive"),
    ({"up": torch.randn(2, 2, 9)}, "same, positive"),
    ({"down": torch.randn(0, 2, 70), "up": torch.randn(0, 2, 9)}, "same, positive"),
    ({"down": torch.randn(3, 129, 70), "up": torch.randn(3, 129, 9)}, "rank 128"),
    ({"ids": torch.zeros(5, dtype=torch.int64)}, "int32"),
    ({"ids": torch.zeros(4, dtype=torch.int32)}, "5 entries"),
    ({"ids": torch.zeros(10, dtype=torch.int32)[::2]}, "contiguous"),
    ({"scale": torch.ones(2)}, "scale"),
    ({"scale": torch.ones(3, dtype=torch.float64)}, "scale"),
    ({"compute": "fp64"}, "compute"),
    ({"out": torch.zeros(5, 8)}, "out must"),
    ({"out": torch.zeros(5, 9, dtype=torch.float64)}, "out must"),
    ({"out": torch.zeros(9, 5).T}, "out must"),
    ({"out": torch.zeros(1, 9).expand(5, 9)}, "do not overlap"),
    ({"prepared": True}, "prepared C"),
])
def test_forward_refusals(change, match):
    args = _forward_args() | change
    with pytest.raises(ValueError, match=match):
        adapted_project_device(**args)


@pytest.mark.parametrize("change,match", [
    ({"dY": torch.randn(4, 9)}, "dY must"),
    ({"dY": torch.randn(5, 0)}, "dY must"),
    ({"dY": torch.randn(5, 8)}, "up must have shape|Ct must have shape"),
    ({"Ct": torch.randn(9, 70)}, "Ct must have shape"),
    ({"hidden": torch.zeros(5, 3)}, "hidden"),
    ({"hidden": torch.zeros(5, 2, dtype=torch.float64)}, "hidden"),
    ({"out": (torch.zeros(3, 2, 69), torch.zeros(3, 2, 9))}, r"out\[0\]"),
    ({"out": (torch.zeros(3, 2, 70), torch.zeros(3, 2, 9, dtype=torch.bfloat16))}, r"out\[1\]"),
    ({"out": (torch.zeros(1, 2, 70).expand(3, 2, 70), torch.zeros(3, 2, 9))}, r"out\[0\]"),
])
def test_backward_refusals(change, match):
    a = _forward_args()
    args = {"dY": torch.randn(5, 9), "X": a["X"], "Ct": torch.randn(70, 9), "down": a["down"], "up": a["up"], "ids": a["ids"],
            "hidden": torch.zeros(5, 2)} | change
    with pytest.raises(ValueError, match=match):
        adapted_project_backward_device(**args)


def test_no_cpu_fallback():
    a = _forward_args()
    with pytest.raises(RuntimeError, match="MI355X"):
        adapted_project_device(*a.values())
    with pytest.raises(RuntimeError, match="MI355X"):
        AdamW([torch.zeros(3)], [torch.zeros(3)])


def test_prepare_bank():
    W = torch.randn(2, 3, 70)
    P = prepare_bank(W, "bf16")
    assert P.shape == (2, 3, 128) and P.dtype == torch.bfloat16 and not P[..., 70:].any()
    assert torch.equal(P[..., :70], W.to(torch.bfloat16))
    assert prepare_bank(P, "bf16") is P
    assert prepare_bank(W, "fp32").shape == (2, 3, 96)


@pytest.mark.parametrize("kw,match", [
    (dict(params=[], grads=[]), "same, positive"),
    (dict(grads=[torch.zeros(3)] * 2), "same, positive"),
    (dict(grads=[torch.zeros(4)]), r"grads\[0\]"),
    (dict(grads=[torch.zeros(3, dtype=torch.float16)]), "float32 or bfloat16"),
    (dict(params=[torch.zeros(3, dtype=torch.bfloat16)]), r"params\[0\]"),
    (dict(params=[torch.zeros(6)[::2]]), r"params\[0\]"),
    (dict(copies=[torch.zeros(3)]), r"copies\[0\]"),
    (dict(copies=[]), "same, positive"),
    (dict(state_bits=16), "32 or 8"),
    (dict(seed=-1), "seed"),
    (dict(betas=(0.9, 1.0)), "betas"),
    (dict(lr=-1.0), "lr"),
    (dict(lr=float("nan")), "lr"),
])
def test_adamw_refusals(kw, match):
    args = {"params": [torch.zeros(3)], "grads": [torch.zeros(3)]} | kw
    with pytest.raises(ValueError, match=match):
        AdamW(args.pop("params"), args.pop("grads"), **args)


def test_adamw_refuses_shared_memory():
    flat = torch.zeros(10)
    for params, grads in (([flat, flat], [torch.zeros(10), torch.zeros(10)]), ([flat[:6], flat[4:]], [torch.zeros(6)] * 2),
                          ([flat], [flat])):
        with pytest.raises(ValueError, match="share memory"):
            AdamW(params, grads)


def test_abi_refuses_before_the_device_is_used():
    lib = nat.load()
    a = 1 << 20  # never read: each call below is refused for another argument
    forward = dict(device=0, X=a, ldx=64, dtype=nat.RP_BF16, n=4, m=64, C=a, p=8, down=a, up=a, G=2, R=4, scale=None, ids=a, Y=a,
                   ldy=8, hidden=None, ws=a, bytes=1 << 20, stream=None)
    for change, code, text in (
            ({"dtype": nat.RP_F64}, nat.RP_ERR_INVALID, b"dtype"), ({"m": 0}, nat.RP_ERR_INVALID, b"bad shape"),
            ({"n": -1}, nat.RP_ERR_INVALID, b"bad shape"), ({"R": 129}, nat.RP_ERR_UNSUPPORTED, b"rank"),
            ({"G": 65536}, nat.RP_ERR_UNSUPPORTED, b"adapters"), ({"ldx": 32}, nat.RP_ERR_INVALID, b"X"),
            ({"X": a + 2}, nat.RP_ERR_INVALID, b"aligned"), ({"ldx": 65}, nat.RP_ERR_INVALID, b"aligned"),
            ({"X": None}, nat.RP_ERR_INVALID, b"NULL X"), ({"up": None}, nat.RP_ERR_INVALID, b"NULL up"),
            ({"ids": None}, nat.RP_ERR_INVALID, b"ids"), ({"ldy": 7}, nat.RP_ERR_INVALID, b"Y"),
            ({"ws": None}, nat.RP_ERR_INVALID, b"workspace"), ({"ws": a + 16}, nat.RP_ERR_INVALID, b"workspace"),
            ({"bytes": 1}, nat.RP_ERR_INVALID, b"workspace")):
        rc = lib.rp_adapt_project_device(*(forward | change).values())
        assert rc == code and text in lib.rp_last_error(), (change, rc, lib.rp_last_error())
    backward = dict(device=0, dY=a, lddy=64, X=a, ldx=64, dtype=nat.RP_BF16, n=4, m=64, p=8, Ct=a, down=a, up=a, G=2, R=4,
                    scale=None, ids=a, hidden=a, dX=a, lddx=64, dd=a, dd_r=64, dd_a=256, du=a, du_r=8, du_a=32, ws=a,
                    bytes=1 << 20, stream=None)
    for change, code, text in (
            ({"lddy": 7}, nat.RP_ERR_INVALID, b"dY"), ({"dY": a + 1}, nat.RP_ERR_INVALID, b"dY"), ({"Ct": None}, nat.RP_ERR_INVALID, b"go together"),
            ({"dX": None}, nat.RP_ERR_INVALID, b"go together"), ({"lddx": 63}, nat.RP_ERR_INVALID, b"dX"),
            ({"dd": None}, nat.RP_ERR_INVALID, b"NULL"), ({"dd_a": 255}, nat.RP_ERR_INVALID, b"strides"),
            ({"du_r": 7}, nat.RP_ERR_INVALID, b"strides"), ({"hidden": None}, nat.RP_ERR_INVALID, b"hidden"),
            ({"bytes": 1}, nat.RP_ERR_INVALID, b"workspace")):
        rc = lib.rp_adapt_gradients_device(*(backward | change).values())
        assert rc == code and text in lib.rp_last_error(), (change, rc, lib.rp_last_error())
    assert lib.rp_adapt_workspace_bytes(nat.RP_BF16, 4, 64, 8, 2, 129, nat.RP_ADAPT_PROJECT) == -1
    h = ctypes.c_void_p()
    one = (ctypes.c_void_p * 1)
    for change, text in (({"T": 0}, b"no tensors"), ({"gt": nat.RP_F64}, b"grad_type"), ({"bits": 4}, b"state_bits"),
                         ({"m": None}, b"NULL state"), ({"m": a + 4}, b"aligned"), ({"w": one(None)}, b"NULL"),
                         ({"w": one(a + 2)}, b"elements"), ({"n": (ctypes.c_int64 * 1)(-1)}, b"bad size")):
        args = dict(device=0, T=1, n=(ctypes.c_int64 * 1)(3), w=one(a), g=one(a), gt=nat.RP_F32, c=None, bits=32, m=a, v=a, ms=None,
                    vs=None, steps=a) | change
        rc = lib.rp_adamw_create(*args.values(), ctypes.byref(h))
        assert rc == nat.RP_ERR_INVALID and text in lib.rp_last_error() and not h, (change, rc, lib.rp_last_error())
    assert lib.rp_adamw_step(None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None, None) == nat.RP_ERR_INVALID
    assert lib.rp_adamw_values(None, None, None, None) == nat.RP_ERR_INVALID
    assert lib.rp_adamw_destroy(None) == nat.RP_OK


def test_workspace_of_every_size():
    lib = nat.load()
    for dtype in (nat.RP_F32, nat.RP_BF16):
        for n in (0, 1, 64, 65, 5000, 10 ** 7):
            for m, p in ((1, 1), (16384, 1024), (100, 70000)):
                for G, R in ((1, 1), (16383, 128)):
                    project, gradients, dx = (lib.rp_adapt_workspace_bytes(dtype, n, m, p, G, R, k) for k in (
                        nat.RP_ADAPT_PROJECT, nat.RP_ADAPT_GRADIENTS, nat.RP_ADAPT_GRADIENTS_DX))
                    assert project >= 0 and dx >= gradients >= 4 * n * R


def test_estimator_without_a_gpu():
    """Parameters, shapes, refusals; the components are the base class's for the same random_state."""
    import pickle

    import numpy as np
    from sklearn.base import clone
    from sklearn.exceptions import NotFittedError

    from randomprojection_amd import AdaptedGaussianProjection
    from randomprojection_amd.gaussian import GaussianRandomProjection

    X = np.random.default_rng(0).standard_normal((20, 33))
    est = AdaptedGaussianProjection(n_components=7, n_adapters=3, rank=2, random_state=5, compute="bf16", state_bits=8)
    with pytest.raises(NotFittedError):
        est.down_
    with pytest.raises(NotFittedError):
        est.transform(X, adapters=np.zeros(20, int))
    assert clone(est).get_params() == est.get_params()
    est.fit(X)
    assert np.array_equal(est.components_, GaussianRandomProjection(n_components=7, random_state=5).fit(X).components_)
    assert est.down_.shape == (3, 2, 33) and est.up_.shape == (3, 2, 7) and not est.up_.any()
    again = pickle.loads(pickle.dumps(est))
    assert np.array_equal(again.down_, est.down_) and np.array_equal(clone(est).fit(X).down_, est.down_)
    for adapters, match in ((np.zeros(19, int), "one whole number"), (np.zeros(20), "one whole number"), (np.full(20, 3), "-1 .. 2"),
                            (np.full(20, -2), "-1 .. 2")):
        with pytest.raises(ValueError, match=match):
            est.transform(X, adapters=adapters)
        with pytest.raises(ValueError, match=match):
            est.partial_fit(X, np.zeros((20, 7)), adapters)
    with pytest.raises(ValueError, match="Y must have shape"):
        est.partial_fit(X, np.zeros((20, 6)), np.zeros(20, int))
    for kw, match in (({"rank": 129}, "rank"), ({"rank": 0}, "rank"), ({"n_adapters": 0}, "n_adapters"), ({"compute": "fp64"}, "compute")):
        with pytest.raises(ValueError, match=match):
            AdaptedGaussianProjection(n_components=7, **kw).fit(X)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="MI355X"):
            est.transform(X, adapters=np.zeros(20, int))


def test_outputs_that_share_memory_with_inputs_are_refused():
    """Columns of one buffer side by side are fine; bytes in common are not."""
    a = _forward_args(n=5, m=64, p=8)
    wide = torch.randn(5, 80)
    for X, out, ok in ((wide[:, :64], wide[:, 64:72], True), (wide[:, 16:], wide[:, 8:16], True), (wide[:, :64], wide[:, 60:68], False),
                       (wide[:, 16:], wide[:, 9:17], False), (wide[:, :64], wide.view(-1)[:40].view(5, 8), False)):
        with pytest.raises(RuntimeError if ok else ValueError, match="MI355X" if ok else "share memory"):
            adapted_project_device(X, a["C"], a["down"], a["up"], a["ids"], out=out)
    with pytest.raises(ValueError, match="share memory"):
        adapted_project_device(a["X"], a["C"], a["down"], a["up"], a["ids"], out=a["C"][:5, :8])
    both = torch.zeros(3, 2, 100)
    grads = lambda x, y: adapted_project_backward_device(torch.randn(5, 8), a["X"], None, a["down"], a["up"], a["ids"],  # noqa: E731
                                                         torch.zeros(5, 2), out=(x, y))
    with pytest.raises(RuntimeError, match="MI355X"):
        grads(both[..., :64], both[..., 64:72])
    for x, y in ((both[..., :64], both[..., 63:71]), (a["down"], both[..., :8]), (both[..., :64], a["up"])):
        with pytest.raises(ValueError, match="share memory"):
            grads(x, y)


def test_adamw_refuses_a_gradient_inside_another_parameter():
    flat = torch.zeros(20)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([flat[:6], flat[6:12]], [flat[12:18], flat[3:9]])
    with pytest.raises(ValueError, match="share memory"):
        AdamW([flat[:4]], [torch.zeros(8).view(torch.bfloat16)[:4]], copies=[flat.view(torch.bfloat16)[6:10]])
    one = torch.zeros(6)
    with pytest.raises(RuntimeError, match="MI355X"):  # a gradient may serve two parameters
        AdamW([flat[:6], flat[6:12]], [one, one])


def test_workspace_for_more_columns_than_the_join_covers():
    lib = nat.load()
    edge = 65535 * 256
    below, above = (lib.rp_adapt_workspace_bytes(nat.RP_BF16, 2, 64, p, 1, 1, nat.RP_ADAPT_PROJECT) for p in (edge, edge + 1))
    assert below > 4 * 2 * edge > above > 0  # partial sums for few rows; none beyond
    assert lib.rp_adapt_workspace_bytes(nat.RP_F32, 1, 2 ** 31 - 100, 8, 1, 1, nat.RP_ADAPT_PROJECT) == -1
