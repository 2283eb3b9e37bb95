"""Adapters and AdamW in calls that the documentation allows: streams of any handle, empty batches, the largest sizes, values
that are not finite, every form of the shrink. Bounds as in test_gpu_adapters.py."""
import pytest
import torch

from test_gpu_adapters import TYPE, check, formulas, make, near

pytestmark = pytest.mark.gpu


def test_default_stream_waits_for_the_current_one():
    """Called under a side stream that still makes the operands, the default stream (handle 0) waits for it."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device
    from randomprojection_amd.gaussian import dense_project_device
    from randomprojection_amd.optim import AdamW

    t = make(700, 333, 100, 6, 8, "bf16", seed=2)
    kw = dict(scale=t["scale"], compute="bf16")

    def run(X, **on):
        Y, h = adapted_project_device(X, t["C"], t["down"], t["up"], t["ids"], return_hidden=True, **kw, **on)
        got = adapted_project_backward_device(t["dY"], X, t["C"].T, t["down"], t["up"], t["ids"], h, **kw, **on)
        w, g = torch.ones(5000, device="cuda"), X.float().view(-1)[:5000]
        opt = AdamW([w], [g], state_bits=8)
        opt.step(**on)
        return [Y, h, *got, w, *opt.state_values(**on), dense_project_device(X, t["C"], compute="bf16", **on)]

    wide = t["X"].double()
    want = run(wide.to(TYPE["bf16"]))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        late = torch.zeros_like(wide)
        torch.cuda._sleep(100_000_000)  # cycles: the copy below comes tens of milliseconds later
        late.copy_(wide)
        got = run(late.to(TYPE["bf16"]), stream=torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_values_behind_a_step_on_another_stream(bits):
    """The states are read out on the stream whose step makes them."""
    from randomprojection_amd.optim import AdamW

    def run(**on):
        g = torch.Generator().manual_seed(1)
        opt = AdamW([torch.zeros(70000, device="cuda")], [torch.randn(70000, generator=g).cuda()], state_bits=bits)
        torch.cuda.synchronize()
        if on:
            with torch.cuda.stream(side):
                torch.cuda._sleep(100_000_000)  # cycles: the step comes tens of milliseconds later
        opt.step(**on)
        got = opt.state_values(**on)
        torch.cuda.synchronize()
        return got

    side = torch.cuda.Stream()
    for a, b in zip(run(stream=side.cuda_stream), run()):
        assert b.any() and torch.equal(a, b)


def test_seed_set_after_fit_waits_for_the_next_fit():
    """Rounding to 8 bits goes by the seed as fitted: two estimators of one history agree bit for bit."""
    from randomprojection_amd import AdaptedGaussianProjection

    g = torch.Generator().manual_seed(1)
    X, T, ids = torch.randn(300, 70, generator=g).numpy(), torch.randn(300, 20, generator=g).numpy(), (torch.arange(300) % 3).numpy()
    kept, changed, other = (AdaptedGaussianProjection(n_components=20, n_adapters=3, rank=4, random_state=3, state_bits=8, seed=s).fit(X)
                            for s in (5, 5, 6))
    changed.set_params(seed=6)
    for _ in range(3):
        for est in (kept, changed, other):
            est.partial_fit(X, T, ids)
    assert (kept.down_ == changed.down_).all() and (kept.up_ == changed.up_).all() and (kept.up_ != other.up_).any()


# Shapes on both sides of the branches that pick a shrink for the forward pass: 16 rows a tile under 512 tiles of 64 rows (32 over rank
# 64), else 64 (32); and 16 again, beside a split product, where there are few tiles of it. The backward pass takes the same branches with
# m and p exchanged. The rank pads to 16, 32, 64 or 128 (f32: its pieces to a multiple of 16).
FORMS = [(32768, 70, 200, 3, 17), (33001, 100, 90, 5, 20), (32768, 65, 66, 3, 32), (33100, 130, 70, 4, 33), (40000, 64, 129, 7, 64), (32799, 200, 65, 2, 48),
         (32767, 70, 200, 3, 20), (32767, 129, 90, 4, 50), (16384, 70, 90, 3, 65), (16383, 100, 70, 2, 128), (35000, 65, 77, 900, 24)]


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", FORMS)
def test_every_form_of_the_shrink(shape, compute):
    """Runs of rows of every length, so that tiles end inside, at and behind a multiple of 16, 32 and 64 rows."""
    n, _, _, G, _ = shape
    g = torch.Generator().manual_seed(sum(shape))
    lengths = torch.randint(1, 300, (n,), generator=g)
    ids = torch.repeat_interleave(torch.randint(-1, G, (n,), generator=g), lengths)[:n]
    check(make(*shape, compute, seed=G, ids=ids), compute, prepared=True)


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("G", [3, 700, 701, 3999, 4000, 16383])
def test_no_rows_whatever_the_number_of_adapters(G, compute):
    """An empty batch: zeros for every adapter, written over what was there; what lies between stays."""
    from randomprojection_amd.adapters import adapted_project_backward_device

    m, p, R = 70, 20, 2
    t = make(0, m, p, G, R, compute)
    bd, bu = torch.full((G, R + 1, m + 3), 7.0, device="cuda"), torch.full((G, R, p + 1), 7.0, device="cuda")
    for Ct in (None, t["C"].T):
        hidden = torch.empty(0, R, device="cuda")
        dX, dd, du = adapted_project_backward_device(t["dY"], t["X"], Ct, t["down"], t["up"], t["ids"], hidden, scale=t["scale"], compute=compute,
                                                     out=(bd[:, :R, :m], bu[..., :p]))
        assert not dd.any() and not du.any() and (Ct is None or dX.shape == (0, m))
        assert bool((bd[:, R] == 7).all()) and bool((bd[..., m:] == 7).all()) and bool((bu[..., p:] == 7).all())
        bd[:, :R, :m], bu[..., :p] = 7.0, 7.0


def test_gradients_of_many_adapters_and_columns():
    """16.8 million blocks of outer products, more than a row of 2^32 threads holds: d_down of 4.3 GB, a few adapters of it with rows."""
    from randomprojection_amd.adapters import adapted_project_backward_device

    n, m, p, G, used = 600, 65536, 64, 16383, [0, 77, 8191, 16382]
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    X, dY, down, up, hidden = r(n, m), r(n, p), r(G, 1, m), r(G, 1, p), r(n, 1)
    ids = torch.tensor(used + [-1], device="cuda", dtype=torch.int32)[torch.arange(n, device="cuda") % 5]
    _, dd, du = adapted_project_backward_device(dY, X, None, down, up, ids, hidden)
    rest = torch.ones(G, dtype=torch.bool, device="cuda")
    rest[used] = False
    for part in torch.nonzero(rest)[:, 0].split(2048):
        assert not dd[part].any() and not du[part].any()
    for a in used:
        at = ids == a
        x, dy, h, u = X[at].double(), dY[at].double(), hidden[at].double(), up[a, 0].double()
        near(dd[a, 0], (dy @ u) @ x, (dy.abs() @ u.abs()) @ x.abs(), n + p + 8)
        near(du[a, 0], h[:, 0] @ dy, h[:, 0].abs() @ dy.abs(), n + 8)


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
def test_product_of_more_tiles_than_a_row_of_the_grid(compute):
    """Over 2^20 tiles: rows of the grid's blocks come after each other. X of 17 GB; rows drawn from all of it."""
    from randomprojection_amd.adapters import adapted_project_device

    n, m, p, G, R = 2 ** 27 + 77, 64 if compute == "bf16" else 32, 1, 3, 1
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=TYPE[compute])  # noqa: E731
    X, C, down, up = r(n, m), r(p, m), r(G, R, m), r(G, R, p)
    ids = (torch.arange(n, device="cuda") * 4 // n - 1).int()
    Y, h = adapted_project_device(X, C, down, up, ids, compute=compute, return_hidden=True)
    rows = torch.cat([torch.randint(0, n, (5000,), generator=g, device="cuda"), torch.arange(n - 200, n, device="cuda"), torch.arange(200, device="cuda")])
    x, a = X[rows].double(), ids[rows].long()
    d, u = (torch.where((a >= 0)[:, None], b[a, 0].double(), 0.0) for b in (down, up))
    hid, size = (x * d).sum(1), (x * d).abs().sum(1)
    near(h[rows, 0], hid, size, m + 8)
    near(Y[rows, 0], x @ C[0].double() + hid * u[:, 0], x.abs() @ C[0].double().abs() + size * u[:, 0].abs(), m + R + 8)


def test_values_of_more_blocks_than_the_grid():
    """Over 2^22 blocks of states in 8 bits: 1.07 billion elements, their values as they are held by an optimizer of the last ones alone."""
    from randomprojection_amd.optim import AdamW

    n, tail = 2 ** 30 + 1000, 3 * 2 ** 18
    g = torch.Generator(device="cuda").manual_seed(1)
    w, grad = torch.zeros(n, device="cuda"), torch.randn(n, device="cuda", generator=g, dtype=torch.bfloat16)
    opt = AdamW([w], [grad], state_bits=8)
    opt.step()
    first = n // 256 * 256 - tail
    alone = AdamW([w[first:]], [grad[first:]], state_bits=8)
    held, own = opt.state_dict(), alone.state_dict()
    alone.load_state_dict({k: (v if k == "steps" else v.view(torch.uint8)[-own[k].numel():].view(v.dtype)) for k, v in held.items()})
    for a, b in zip(opt.state_values(), alone.state_values()):
        assert a.numel() == held["exp_avg"].numel() and b.any() and torch.equal(a[-b.numel():], b)
        middle = a[2 ** 29:2 ** 29 + 10 ** 6].double()
        assert bool(middle.any()) and bool(torch.isfinite(middle).all())


@pytest.mark.parametrize("compute", ["bf16", "fp32"])
@pytest.mark.parametrize("n,m,p,R", [(40, 70, 90, 6), (700, 70, 90, 6), (20000, 70, 90, 6), (20000, 130, 150, 40), (35000, 64, 50, 20)])
def test_infinities_are_those_of_the_formulas(n, m, p, R, compute):
    """An infinity in an operand gives what the formulas give, an infinity or a NaN, whatever the number of rows. All values are small
    whole numbers and halves, whose products and sums are exact in f32, and whose pieces of fewer bits are zeros mostly."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device

    G, inf = 6, float("inf")
    g = torch.Generator().manual_seed(n)
    pick = lambda *s: torch.randint(1, 3, s, generator=g).float() * (torch.randint(0, 2, s, generator=g) * 2 - 1)  # noqa: E731
    t = {"X": pick(n, m), "C": pick(p, m), "down": pick(G, R, m), "up": pick(G, R, p), "dY": pick(n, p)}
    t["up"][2, 1, 5], t["up"][3, R - 1, 7], t["up"][4, 0, p - 1], t["down"][1, 2, 9], t["down"][2, 0, m - 1] = inf, -inf, inf, inf, -inf
    t["X"][8, 33], t["X"][13, 0], t["X"][n - 1, 1], t["dY"][22, 5], t["dY"][n - 3, p - 1] = inf, -inf, inf, -inf, inf  # of adapters 0 and 5, ..
    t = {k: v.to(TYPE[compute]) for k, v in t.items()}
    t["scale"] = torch.tensor([1.0, 0.5, 2.0, -1.0, 0.0, 1.5])
    t["ids"] = (torch.arange(n) % (G + 1) - 1).int()
    u = {k: v.cuda() for k, v in t.items()}
    kw = dict(scale=u["scale"], compute=compute)
    Y, h = adapted_project_device(u["X"], u["C"], u["down"], u["up"], u["ids"], return_hidden=True, **kw)
    got = dict(zip(("dX", "d_down", "d_up"), adapted_project_backward_device(u["dY"], u["X"], u["C"].T, u["down"], u["up"], u["ids"], h, **kw)))
    got |= {"Y": Y, "hidden": h}
    want, _ = formulas(t, h.cpu())
    for k, x in got.items():
        a, b = x.cpu(), want[k].to(x.dtype)
        same = (a == b) | (a.isnan() & b.isnan())
        assert same.all(), (k, torch.nonzero(~same)[:4].tolist(), a[~same][:4], b[~same][:4])
        assert b.isinf().any() and b.isfinite().any(), k


@pytest.mark.parametrize("kind", ["steady", "random", "one burst"])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.99), (0.95, 0.95)])
def test_small_gradients_beside_large_ones_in_8_bits(betas, kind):
    """Elements whose gradients are far below their block's largest: the least code of m is taken only where B root covers it, and steps
    stay near what AdamW can make.

    Each step's codes are compared with m and the root in f32 from the values held before it: an m under the least code l is held as 0 where
    l > B root, as 0 or l elsewhere; other m as one of the codes on its two sides (1e-5 aside, for the roundings in B root).
    A steady gradient under l, which only grows while the block's largest m does, leaves m in {0, l}: b1 l + (1 - b1) |g| < l. l is held where it
    is at most B root, a code of the root is at least 8/9 of it, and root' >= sqrt(b2) root_held, sqrt(1 - b2) |g|: so
    |m'| / root' <= b1 B (9/8) / sqrt(b2) + (1 - b1) / sqrt(1 - b2). Roots too small for 8/9 (under 2^-30 of the largest) never hold l. The
    step is lr sqrt(1 - b2^t) / (1 - b1^t) times that."""
    from randomprojection_amd.optim import AdamW

    (b1, b2), lr, steps, ratios = betas, 1e-3, 600, [1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12]
    B = (1 - b1) / ((1 - b2) * (1 - b1 ** 2 / b2)) ** 0.5
    most = (b1 * B * 9 / 8 / b2 ** 0.5 + (1 - b1) / (1 - b2) ** 0.5) * max((1 - b2 ** t) ** 0.5 / (1 - b1 ** t) for t in range(1, steps + 1))
    scale = torch.tensor(ratios, device="cuda")[:, None].expand(-1, 1024).clone()
    scale[:, ::256] = 1.0  # one in each block of 256
    grad, w = scale.clone(), torch.zeros_like(scale)
    opt = AdamW(list(w), list(grad), lr=lr, betas=betas, eps=0.0, weight_decay=0.0, state_bits=8, seed=3)
    rand = torch.Generator(device="cuda").manual_seed(2)
    largest, before = torch.zeros_like(w), w.clone()
    m0, r0 = opt.state_values()
    refused = taken = 0
    for t in range(steps):
        if kind == "random":
            grad.copy_(scale * torch.randn(scale.shape, device="cuda", generator=rand))
        elif kind == "one burst" and t == 300:
            grad.mul_(torch.where(scale < 1, 30.0, 1.0))
        elif kind == "one burst" and t == 301:
            grad.copy_(scale)
        opt.step()
        largest = torch.maximum(largest, (w - before).abs())
        before.copy_(w)
        g = grad.view(-1)
        m, root = (m0 * b1 + g * (1 - b1)).abs(), (r0 * r0 * b2 + g * g * (1 - b2)).sqrt()
        least = ((m.view(28, 256).amax(1).view(torch.int32) >> 23) - 16 << 23).view(torch.float32).repeat_interleave(256)  # 2^-16 of its binade
        m0, r0 = opt.state_values()
        held, under = m0.abs(), m < least * (1 - 1e-5)
        refuse, take = under & (least > B * root * (1 + 1e-5)), under & (least < B * root * (1 - 1e-5))
        assert not held[refuse].any() and ((held == 0) | (held == least))[under].all()
        assert ((held - m).abs() <= torch.maximum(least, m / 8)).all()
        refused, taken = refused + int((refuse & (m > 0)).sum()), taken + int((held[take] > 0).sum())
    assert refused and taken and torch.isfinite(w).all()
    if kind == "steady":
        small = scale[:, 1] <= 1e-7
        # 1e-5 for the roundings in the step, and half a step of w for its own
        assert (largest.amax(1) <= lr * most * (1 + 1e-5) + w.abs().amax(1) * 2.0 ** -24)[small].all(), (largest.amax(1) / lr, most)
        assert (w < 0).all()  # each moves against its gradient, the small ones too


def test_least_code_where_gradients_bound_nothing():
    """b1^2 >= b2: any m can lie beside any root, so every m under the least code is rounded at random."""
    from randomprojection_amd.optim import AdamW

    g = torch.full((4096,), 1e-6, device="cuda")
    g[::256] = 1.0
    opt = AdamW([torch.zeros(4096, device="cuda")], [g], betas=(0.95, 0.9), state_bits=8, lr=1e-3)
    opt.step()
    held = opt.state_values()[0]
    small = g < 1
    # m = 5e-8, the least code 2^-16 of the binade of 0.05, 4.8e-7: about a tenth of 4080 are held as it (standard deviation 19)
    least = 2.0 ** -5 * 2.0 ** -16
    assert ((held == 0) | (held == least))[small].all() and 300 < int((held[small] > 0).sum()) < 560
    assert torch.isfinite(opt.params[0]).all()
