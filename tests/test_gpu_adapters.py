"""Adapters beside the dense projection, forward and backward, against 64 bits.

Bounds: a sum of K exact products held in f32 is off by at most K 2^-24 of the sum of their magnitudes
whatever its order; 2^-23 is allowed for each step, in case the matrix units cut off where they round. So every
output is compared element by element with ``steps * 2^-23 * (the same formula over magnitudes)``; dX in bf16
adds half a step, 2^-8 of its value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -23
TYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


def make(n, m, p, G, R, compute, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"X": r(n, m), "C": r(p, m) * p ** -0.5, "down": r(G, R, m) * m ** -0.5, "up": r(G, R, p) * R ** -0.5, "dY": r(n, p)}
    t = {k: v.to(TYPE[compute]).cuda() for k, v in t.items()}
    t["scale"] = (torch.rand(G, generator=g) * 2 - 0.5).cuda()
    if ids is None:
        ids = torch.randint(-1, G, (n,), generator=g)
    t["ids"] = torch.as_tensor(ids, dtype=torch.int32).cuda()
    return t


def formulas(t, hidden=None):
    """Y, hidden and the gradients in 64 bits, and each one's magnitude."""
    d = {k: v.double() for k, v in t.items() if k != "ids"}
    ids, G = t["ids"].long(), t["down"].shape[0]

    def compute(d, hidden):
        n, R = d["X"].shape[0], d["down"].shape[1]
        o = {"Y": d["X"] @ d["C"].T, "hidden": d["X"].new_zeros(n, R), "dX": d["dY"] @ d["C"],
             "d_down": torch.zeros_like(d["down"]), "d_up": torch.zeros_like(d["up"])}
        for g in range(G):
            at = torch.nonzero(ids == g)[:, 0]
            x, dy, s = d["X"][at], d["dY"][at], d["scale"][g]
            h = x @ d["down"][g].T
            o["hidden"][at] = h
            o["Y"][at] += s * (h @ d["up"][g])
            tt = s * (dy @ d["up"][g].T)
            o["dX"][at] += tt @ d["down"][g]
            o["d_down"][g] = tt.T @ x
            o["d_up"][g] = s * ((h if hidden is None else hidden[at]).T @ dy)
        return o

    hidden = None if hidden is None else hidden.double()
    return compute(d, hidden), compute({k: v.abs() for k, v in d.items()}, None if hidden is None else hidden.abs())


def near(got, want, size, steps, half=0.0):
    err = (got.double() - want).abs()
    bound = steps * E * size + half * want.abs() * (1 + 1e-3) + 1e-30
    bad = err > bound
    assert torch.isfinite(got).all() and not bad.any(), (int(bad.sum()), float((err / bound).max()))


def check(t, compute, prepared=False, **kw):
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device, prepare_bank

    (n, m), p, R = t["X"].shape, t["C"].shape[0], t["down"].shape[1]
    ops = {"C": t["C"], "Ct": t["C"].T, "down": t["down"], "up": t["up"]}
    if prepared:
        ops = {k: prepare_bank(v, compute) for k, v in ops.items()}
    Y, hidden = adapted_project_device(t["X"], ops["C"], ops["down"], ops["up"], t["ids"], scale=t["scale"], compute=compute,
                                       return_hidden=True, prepared=prepared, **kw)
    dX, dd, du = adapted_project_backward_device(t["dY"], t["X"], ops["Ct"], ops["down"], ops["up"], t["ids"], hidden,
                                                 scale=t["scale"], compute=compute, prepared=prepared)
    none, dd2, du2 = adapted_project_backward_device(t["dY"], t["X"], None, ops["down"], ops["up"], t["ids"], hidden,
                                                     scale=t["scale"], compute=compute, prepared=prepared)
    want, size = formulas(t, hidden)
    assert Y.shape == (n, p) and hidden.shape == (n, R) and dX.shape == (n, m) and dX.dtype == TYPE[compute]
    near(Y, want["Y"], size["Y"], m + R + 8)
    near(hidden, want["hidden"], size["hidden"], m + 8)
    near(dX, want["dX"], size["dX"], p + R + 8, 2.0 ** -8 if compute == "bf16" else 0.0)
    near(dd, want["d_down"], size["d_down"], n + p + 8)
    near(du, want["d_up"], size["d_up"], n + 8)
    assert none is None and torch.equal(dd, dd2) and torch.equal(du, du2)
    return Y, hidden, dX, dd, du


SHAPES = [(1, 64, 1, 1, 1), (1, 4096, 1024, 8, 16), (2, 65, 3, 2, 3), (16, 128, 16, 4, 16), (17, 100, 33, 20, 5),
          (63, 640, 130, 64, 8), (64, 2048, 257, 3, 64), (65, 511, 64, 7, 17), (129, 1000, 129, 6, 33), (300, 4096, 200, 4, 8),
          (257, 192, 129, 5, 128), (515, 320, 1024, 1, 32), (1000, 64, 700, 300, 4), (2049, 256, 300, 3, 16), (4100, 384, 72, 24, 64)]


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formulas(shape, compute):
    check(make(*shape, compute, seed=sum(shape)), compute)


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["none", "one", "last", "runs", "alternating", "outside"])
@pytest.mark.parametrize("n", [40, 333])
def test_rows_and_adapters(n, kind, compute):
    """No row with an adapter, all with one, runs of every length, neighbours that differ, ids outside the range."""
    G = 9
    ids = {"none": np.full(n, -1), "one": np.full(n, 4), "last": np.where(np.arange(n) == n - 1, G - 1, -1),
           "runs": np.repeat(np.arange(n) % (G + 1) - 1, np.arange(n))[:n], "alternating": np.arange(n) % G,
           "outside": np.array([-1, G, G + 1, 2 ** 31 - 1, -2 ** 31, 3])[np.arange(n) % 6]}[kind]
    t = make(n, 320, 150, G, 12, compute, seed=n, ids=ids)
    _, hidden, _, dd, du = check(t, compute)
    with_rows = set(int(i) for i in ids) & set(range(G))
    for g in range(G):
        assert bool(dd[g].any()) == bool(du[g].any()) == (g in with_rows)
    assert not hidden[torch.as_tensor((ids < 0) | (ids >= G)).cuda()].any()


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [30, 700])
def test_not_finite_stays_where_it_is(n, compute):
    """A NaN or an infinity in one row, or in an adapter, reaches that row and that adapter's rows and gradients only."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    G = 5
    t = make(n, 200, 90, G, 6, compute, seed=3, ids=np.arange(n) % (G + 1) - 1)

    def run(t):
        Y, h = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute, return_hidden=True)
        return (Y, h, *adapted_project_backward_device(t["dY"], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h, scale=t["scale"],
                                                       compute=compute))

    clean = run(t)
    for value in (float("nan"), float("inf"), -float("inf")):
        u = dict(t, X=t["X"].clone(), dY=t["dY"].clone())
        u["X"][7, 33] = value  # row 7 has adapter 0
        u["dY"][12, 5] = value  # row 12 has none
        got = run(u)
        rows = torch.ones(n, dtype=torch.bool, device="cuda")
        rows[[7, 12]] = False
        for k in range(3):
            assert torch.equal(got[k][rows], clean[k][rows]), k
        assert not torch.isfinite(got[0][7]).any() and not torch.isfinite(got[2][12]).any()
        for k in (3, 4):
            assert torch.equal(got[k][1:], clean[k][1:])
        u = dict(t, down=t["down"].clone(), up=t["up"].clone())
        u["down"][2] = value
        u["up"][2] = value
        got = run(u)
        others = t["ids"] != 2
        for k in range(3):
            assert torch.equal(got[k][others], clean[k][others]), k
        for k in (3, 4):
            assert torch.equal(got[k][[0, 1, 3, 4]], clean[k][[0, 1, 3, 4]])
    u = dict(t, scale=torch.full_like(t["scale"], float("nan")))
    none = t["ids"] < 0
    assert torch.equal(run(u)[0][none], clean[0][none])


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [33, 600])
def test_strides_and_outputs(n, compute):
    """Rows inside wider buffers, outputs inside wider ones (what lies between stays), prepared operands, other types cast."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    t = make(n, 256, 130, 4, 10, compute, seed=5)
    Y, h, dX, dd, du = check(t, compute)
    assert all(torch.equal(a, b) for a, b in zip(check(t, compute, prepared=True), (Y, h, dX, dd, du)))
    wide = torch.full((n, 400), float("nan"), device="cuda", dtype=TYPE[compute])
    wide[:, 64:320] = t["X"]
    buf = torch.full((n, 200), 7.0, device="cuda")
    got = adapted_project_device(wide[:, 64:320], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute, out=buf[:, 3:133])
    assert torch.equal(got, Y) and bool((buf[:, :3] == 7).all()) and bool((buf[:, 133:] == 7).all())
    wide[:, 65:321] = t["X"]  # rows that are not aligned
    assert torch.equal(adapted_project_device(wide[:, 65:321], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute), Y)
    columns = t["X"].T.contiguous().T
    assert torch.equal(adapted_project_device(columns, t["C"].T.contiguous().T, t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute), Y)
    bd, bu = torch.full((4, 11, 300), 7.0, device="cuda"), torch.full((4, 10, 131), 7.0, device="cuda")
    dyw = torch.full((n, 192), float("nan"), device="cuda", dtype=TYPE[compute])
    dyw[:, :130] = t["dY"]
    got = adapted_project_backward_device(dyw[:, :130], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h, scale=t["scale"], compute=compute,
                                          out=(bd[:, :10, :256], bu[..., :130]))
    assert torch.equal(got[0], dX) and torch.equal(bd[:, :10, :256], dd) and torch.equal(bu[..., :130], du)
    assert bool((bd[:, 10:] == 7).all()) and bool((bd[..., 256:] == 7).all()) and bool((bu[..., 130:] == 7).all())
    other = {k: t[k].double() for k in ("X", "C", "down", "up")}
    assert torch.equal(adapted_project_device(*other.values(), t["ids"], scale=t["scale"], compute=compute), Y)
    one = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], compute=compute)
    assert torch.equal(one, adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], scale=torch.ones(4, device="cuda"), compute=compute))


def test_no_rows():
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    t = make(0, 100, 20, 3, 4, "bf16")
    Y, h = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], compute="bf16", return_hidden=True)
    assert Y.shape == (0, 20) and h.shape == (0, 4)
    dX, dd, du = adapted_project_backward_device(t["dY"], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h, compute="bf16")
    assert dX.shape == (0, 100) and not dd.any() and not du.any() and dd.shape == (3, 4, 100) and du.shape == (3, 4, 20)


@pytest.mark.parametrize("n", [50, 150])
def test_gradients_against_differences(n):
    """Y is linear in X, in up and in down each: a difference of any length gives the derivative of <dY, Y> but for rounding."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    t = make(n, 192, 100, 4, 6, "fp32", seed=8)
    Y, h = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], return_hidden=True)
    grads = dict(zip(("X", "down", "up"), adapted_project_backward_device(t["dY"], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h, scale=t["scale"])))
    _, size = formulas(t)
    g = torch.Generator(device="cuda").manual_seed(9)
    for k, grad in grads.items():
        step = torch.randn(t[k].shape, device="cuda", generator=g)
        Y2 = adapted_project_device(*(dict(t, **{k: t[k] + step})[j] for j in ("X", "C", "down", "up")), t["ids"], scale=t["scale"])
        moved, said = float((t["dY"].double() * (Y2.double() - Y.double())).sum()), float((grad.double() * step.double()).sum())
        # both Y are off by (m + R + 8) steps of their magnitude, the step itself by half a one
        u = formulas(dict(t, **{k: t[k].abs() + step.abs()}))[1]["Y"]
        allowed = float((t["dY"].double().abs() * (size["Y"] + 3 * u)).sum()) * 220 * E
        assert abs(moved - said) < allowed < 0.4 * float(grad.double().norm()), (k, moved, said, allowed)


@pytest.mark.parametrize("n", [20, 700])
def test_other_stream_graph_and_repeats(n):
    """The same bits on another stream, twice in a row, and from a graph that is replayed with other inputs between."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device, prepare_bank

    t = make(n, 333, 100, 6, 8, "bf16", seed=2)
    other = make(n, 333, 100, 6, 8, "bf16", seed=4)
    ops = [prepare_bank(t[k], "bf16") for k in ("C", "down", "up")]
    Ct = prepare_bank(t["C"].T, "bf16")

    def run(X, dY, ids, **kw):
        Y, h = adapted_project_device(X, *ops, ids, scale=t["scale"], compute="bf16", prepared=True, return_hidden=True, **kw)
        return (Y, h, *adapted_project_backward_device(dY, X, Ct, *ops[1:], ids, h, scale=t["scale"], compute="bf16", prepared=True, **kw))

    want, want2 = run(t["X"], t["dY"], t["ids"]), run(other["X"], other["dY"], other["ids"])
    assert all(torch.equal(a, b) for a, b in zip(run(t["X"], t["dY"], t["ids"]), want))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    Y, h = adapted_project_device(t["X"], *ops, t["ids"], scale=t["scale"], compute="bf16", prepared=True, return_hidden=True, stream=side.cuda_stream)
    side.synchronize()
    got = adapted_project_backward_device(t["dY"], t["X"], Ct, *ops[1:], t["ids"], h, scale=t["scale"], compute="bf16", prepared=True, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((Y, h, *got), want))
    with torch.cuda.stream(side):
        got = run(t["X"], t["dY"], t["ids"])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    X, dY, ids = (t[k].clone() for k in ("X", "dY", "ids"))
    graphs = []
    for _ in range(2):
        run(X, dY, ids)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(X, dY, ids)
        graphs.append((g, out))
    for k in range(4):
        src, expect = ((t, want), (other, want2))[k % 2]
        for name, buf in (("X", X), ("dY", dY), ("ids", ids)):
            buf.copy_(src[name])
        for g, out in graphs:  # one behind the other, over one set of inputs
            g.replay()
        run(t["X"], t["dY"], t["ids"])
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, expect)), k


def test_many_adapters_and_wide_rows():
    """More adapters than rows in a tile, a row count past a block, far offsets in the banks."""
    t = make(777, 4096, 64, 2000, 3, "bf16", seed=11)
    check(t, "bf16")


# products of few tiles are split over the contraction where that takes less time than the tiles leave idle, others whole, in tiles of 128 or of
# 256 rows and columns, whichever takes less time; over 8192 rows or 700 adapters are grouped by several blocks; from 32768 rows on (16384 over
# rank 64) the shrink takes more rows at a time
LARGE = [(2049, 1100, 1150, 7, 40), (3001, 1030, 700, 3, 128), (2050, 4100, 1090, 700, 1), (4100, 2950, 3000, 11, 17), (9001, 200, 2000, 5, 64),
         (8193, 64, 64, 701, 4), (8192, 100, 130, 700, 2), (33000, 96, 1040, 3, 9), (17000, 72, 1101, 2, 100), (20000, 128, 300, 5000, 2),
         (300, 70, 65, 16383, 1)]


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", LARGE)
def test_large_against_the_formulas(shape, compute):
    G = shape[3]
    g = torch.Generator().manual_seed(sum(shape))
    # runs of rows, as requests have, but for a third of them
    ids = torch.repeat_interleave(torch.randint(-1, G, (shape[0] // 40 + 1,), generator=g), 40)[:shape[0]]
    ids = torch.where(torch.rand(shape[0], generator=g) < 0.33, torch.randint(-1, G, (shape[0],), generator=g), ids)
    check(make(*shape, compute, seed=G, ids=ids), compute, prepared=True)


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(2500, 900, 1001, 5, 6), (4200, 2880, 2999, 4, 20)])
def test_large_outputs_keep_to_their_rows(shape, compute):
    """Not finite values stay where they are, and what lies around strided outputs stays, where whole tiles are multiplied too."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    n, m, p, G, R = shape
    t = make(*shape, compute, seed=7, ids=np.arange(n) % (G + 1) - 1)
    buf = torch.full((n + 5, p + 9), 7.0, device="cuda")

    def run(t, out=None):
        Y, h = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute, return_hidden=True, out=out)
        return (Y, h, *adapted_project_backward_device(t["dY"], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h, scale=t["scale"],
                                                       compute=compute))

    clean = run(t)
    again = run(t, out=buf[2:n + 2, 3:p + 3])
    assert all(torch.equal(a, b) for a, b in zip(clean, again))
    buf[2:n + 2, 3:p + 3] = 7
    assert bool((buf == 7).all())
    for value in (float("nan"), -float("inf")):
        u = dict(t, X=t["X"].clone(), dY=t["dY"].clone(), down=t["down"].clone(), up=t["up"].clone())
        u["X"][0, 33] = value  # no adapter
        u["dY"][n - 1, 5] = value
        u["down"][2], u["up"][2] = value, value
        got = run(u)
        rows = t["ids"] != 2
        rows[0] = rows[n - 1] = False
        for k in range(3):
            assert torch.equal(got[k][rows], clean[k][rows]), k
        whole = [g for g in range(G) if g not in (2, int(t["ids"][n - 1]))]
        for k in (3, 4):
            assert torch.equal(got[k][whole], clean[k][whole])


def test_large_graph_on_another_stream():
    """A captured forward and backward pass of whole tiles, replayed with other inputs between, while eager calls run beside it."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device, prepare_bank

    shape = (9000, 1000, 700, 6, 8)
    t, other = make(*shape, "bf16", seed=2), make(*shape, "bf16", seed=4)
    ops, Ct = [prepare_bank(t[k], "bf16") for k in ("C", "down", "up")], prepare_bank(t["C"].T, "bf16")

    def run(X, dY, ids):
        Y, h = adapted_project_device(X, *ops, ids, scale=t["scale"], compute="bf16", prepared=True, return_hidden=True)
        return (Y, h, *adapted_project_backward_device(dY, X, Ct, *ops[1:], ids, h, scale=t["scale"], compute="bf16", prepared=True))

    want = [run(s["X"], s["dY"], s["ids"]) for s in (t, other)]
    X, dY, ids = (t[k].clone() for k in ("X", "dY", "ids"))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = run(X, dY, ids)
    for k in range(4):
        for name, b in (("X", X), ("dY", dY), ("ids", ids)):
            b.copy_((t, other)[k % 2][name])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        beside = run(t["X"], t["dY"], t["ids"])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 2])) and all(torch.equal(a, b) for a, b in zip(beside, want[0])), k


def test_offsets_past_32_bits():
    """X of 5.2 GB, a bank's row and its gradients by rows and columns drawn from all of them."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    n, m, p, G, R = 40000, 65536, 70, 2, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    X, C, down, up, dY = r(n, m), r(p, m), r(G, R, m), r(G, R, p), r(n, p)
    ids = (torch.arange(n, device="cuda") * 3 // n - 1).int()
    Y, h = adapted_project_device(X, C, down, up, ids, compute="bf16", return_hidden=True)
    dX, dd, du = adapted_project_backward_device(dY, X, C.T, down, up, ids, h, compute="bf16")
    rows = torch.tensor([0, 1, 13333, 16384, 26666, 26667, 32767, 32768, 39998, 39999], device="cuda")
    cols = torch.tensor([0, 1, 32767, 32768, 65534, 65535], device="cuda")
    c, d, u = C.double(), down.double(), up.double()
    for i in rows.tolist():
        x, y, a = X[i].double(), dY[i].double(), int(ids[i])
        hid = d[a] @ x if a >= 0 else torch.zeros(R, device="cuda", dtype=torch.double)
        size_h = d[a].abs() @ x.abs() if a >= 0 else hid
        near(h[i], hid, size_h, m + 8)
        near(Y[i], c @ x + (hid @ u[a] if a >= 0 else 0), c.abs() @ x.abs() + (size_h @ u[a].abs() if a >= 0 else 0), m + R + 8)
        tt = u[a] @ y if a >= 0 else hid
        size_t = u[a].abs() @ y.abs() if a >= 0 else hid
        near(dX[i], y @ c + (tt @ d[a] if a >= 0 else 0), y.abs() @ c.abs() + (size_t @ d[a].abs() if a >= 0 else 0), p + R + 8, 2.0 ** -8)
    for a in range(G):
        at = ids == a
        y, x, hid = dY[at].double(), X[at][:, cols].double(), h[at].double()
        near(dd[a][:, cols], (u[a] @ y.T) @ x, (u[a].abs() @ y.abs().T) @ x.abs(), n + p + 8)
        near(du[a], hid.T @ y, hid.abs().T @ y.abs(), n + 8)


def test_more_columns_than_the_join_covers():
    """Two rows by 17 million components, C of 2.2 GB."""
    from randomprojection_amd.adapters import adapted_project_device

    n, m, p = 2, 64, 17_000_000
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    X, C, down, up = r(n, m), r(p, m), r(1, 1, m), r(1, 1, p)
    Y = adapted_project_device(X, C, down, up, torch.tensor([0, -1], dtype=torch.int32, device="cuda"), compute="bf16")
    for part in (slice(0, 1000), slice(65535 * 256 - 500, 65535 * 256 + 500), slice(p - 1000, p)):
        x, c, u = X.double(), C[part].double(), up[0, 0, part].double()
        hid = x[0] @ down[0, 0].double()
        near(Y[0, part], x[0] @ c.T + hid * u, x[0].abs() @ c.abs().T + x[0].abs() @ down[0, 0].double().abs() * u.abs(), m + 9)
        near(Y[1, part], x[1] @ c.T, x[1].abs() @ c.abs().T, m + 9)


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (70, 7, 5, 3, 4), (33, 3, 2, 2, 2), (200, 9, 15, 3, 16), (90, 8, 4, 2, 3), (513, 5, 3, 4, 17), (9000, 4, 130, 3, 2),
                                   (600, 129, 127, 2, 9), (700, 121, 1100, 3, 70), (20000, 15, 9, 5, 3)])
def test_narrow_and_odd_widths(shape, compute):
    """Rows shorter than a lane's loads, and rows that end inside one, lying between others that are not numbers."""
    n, m, p, G, R = shape
    t = make(*shape, compute, seed=sum(shape))
    want = check(t, compute)
    for k, w, left in (("X", m, 3), ("dY", p, 5)):
        wide = torch.full((n + 1, w + 11), float("nan"), device="cuda", dtype=TYPE[compute])
        inside = wide.view(-1)[left:left + n * (w + 11)].view(n, w + 11)[:, :w]
        inside.copy_(t[k])
        t[k] = inside
    assert all(torch.equal(a, b) for a, b in zip(check(t, compute), want))


@pytest.mark.parametrize("n,G", [(300001, 7), (270000, 1000), (100000, 16383), (12289, 701)])
def test_grouping_of_many_rows(n, G):
    """Exact whole numbers: each row gets its own adapter's part, each adapter the sum over its own rows."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    g = torch.Generator().manual_seed(n)
    ids = torch.randint(-2, G + 2, (n,), generator=g, dtype=torch.int32).cuda()
    X = (torch.arange(n) % 5 - 2).float()[:, None].cuda()
    a = torch.arange(G, device="cuda").float()[:, None, None]
    down, up, C = a % 127 + 1, a // 127 + 1, torch.ones(1, 1, device="cuda")
    Y, h = adapted_project_device(X, C, down, up, ids, return_hidden=True)
    ok = (ids >= 0) & (ids < G)
    at = torch.where(ok, ids, 0).long()
    d, u = torch.where(ok, down[at, 0, 0], 0), torch.where(ok, up[at, 0, 0], 0)
    assert torch.equal(h, X * d[:, None]) and torch.equal(Y, X + X * (d * u)[:, None])
    _, dd, du = adapted_project_backward_device(torch.ones_like(Y), X, None, down, up, ids, h)
    want = torch.zeros(G, dtype=torch.float64, device="cuda").index_add_(0, at, torch.where(ok, X[:, 0], 0).double())
    assert torch.equal(dd[:, 0, 0].double(), want * up[:, 0, 0]) and torch.equal(du[:, 0, 0].double(), want * down[:, 0, 0])


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("G", [1, 3, 800, 16383])
@pytest.mark.parametrize("n,m,p,R", [(1, 63, 65, 1), (2, 4097, 7, 20), (16, 31, 1029, 16), (17, 127, 129, 3), (33, 2050, 61, 33), (64, 999, 1001, 16)])
def test_few_odd_rows(n, m, p, R, G, compute):
    """Up to 64 rows that end inside a line, between others that are not numbers, in every order of their adapters."""
    if G == 16383 and R > 16:
        R = 2
    g = torch.Generator().manual_seed(n + G)
    ids = torch.randint(-1, min(G, 9), (n,), generator=g) * max(1, (G - 1) // 9)
    t = make(n, m, p, 1 if G == 1 else G, R, compute, seed=n, ids=ids)
    for k, w, left in (("X", m, 1), ("dY", p, 3)):
        wide = torch.full((n + 1, w + 6), float("nan"), device="cuda", dtype=TYPE[compute])
        inside = wide.view(-1)[left:left + n * (w + 6)].view(n, w + 6)[:, :w]
        inside.copy_(t[k])
        t[k] = inside
    if G <= 3:
        check(t, compute)
        return
    # many adapters: the few that have rows in 64 bits, the others' gradients zero
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    used = sorted(set(int(i) for i in ids if 0 <= i < G))
    small = dict(t, down=t["down"][used], up=t["up"][used], scale=t["scale"][used],
                 ids=torch.tensor([used.index(int(i)) if int(i) in used else -1 for i in ids], dtype=torch.int32, device="cuda"))
    if not used:
        return
    Y, h, dX, dd, du = check(small, compute)
    Y2, h2 = adapted_project_device(t["X"], t["C"], t["down"], t["up"], t["ids"], scale=t["scale"], compute=compute, return_hidden=True)
    dX2, dd2, du2 = adapted_project_backward_device(t["dY"], t["X"], t["C"].T, t["down"], t["up"], t["ids"], h2, scale=t["scale"], compute=compute)
    assert torch.equal(Y, Y2) and torch.equal(h, h2) and torch.equal(dX, dX2)
    assert torch.equal(dd2[used], dd) and torch.equal(du2[used], du)
    rest = torch.ones(G, dtype=torch.bool, device="cuda")
    rest[used] = False
    assert not dd2[rest].any() and not du2[rest].any()


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(9000, 64, 50, 4, 40), (3000, 700, 64, 3, 128), (40000, 60, 33, 5, 9), (50000, 1000, 64, 6, 16), (700, 5000, 3, 9, 7), (45000, 63, 1, 2, 1)])
def test_narrow_results(shape, compute):
    """Up to 64 columns of Y or of dX."""
    g = torch.Generator().manual_seed(shape[0])
    ids = torch.repeat_interleave(torch.randint(-1, shape[3], (shape[0] // 50 + 1,), generator=g), 50)[:shape[0]]
    check(make(*shape, compute, seed=shape[1], ids=ids), compute)
