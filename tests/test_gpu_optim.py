"""AdamW over many tensors, against 64 bits and, for the states in 8 bits, against their definition in whole numbers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24  # half a step of f32
SIZES = [1, 255, 256, 257, 1023, 1024, 1025, 5000, 3, 0, 2048, 70000]
NUMBERS = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
M32 = 0xFFFFFFFF


def make(sizes, bits, grads=torch.float32, copies=True, seed=0, offset=0, shuffle=False):
    """An optimizer over tensors of these sizes; ``offset`` elements past an aligned address."""
    from randomprojection_amd.optim import AdamW

    g = torch.Generator().manual_seed(seed)
    r = lambda n, dt: torch.cat([torch.zeros(offset), torch.randn(n, generator=g)]).to(dt).cuda()[offset:]  # noqa: E731
    params = [r(n, torch.float32) for n in sizes]
    gs = [r(n, grads) * (10.0 ** (i % 5 - 3)) for i, n in enumerate(sizes)]
    gs = [torch.cat([x.new_zeros(offset), x])[offset:] for x in gs]
    cs = [torch.full((n + offset,), 7.0, dtype=torch.bfloat16, device="cuda")[offset:] for n in sizes] if copies else None
    return AdamW(params, gs, state_bits=bits, copies=cs, seed=1234567890123, **NUMBERS)


def parts(opt, flat):
    at, got = 0, []
    for p in opt.params:
        got.append(flat[at:at + p.numel()])
        at += -(-p.numel() // 256) * 256
    return got


def mix(x):
    x = x ^ (x >> np.uint64(16))
    x = x * np.uint64(0x9E3779B1) & np.uint64(M32)
    x = x ^ (x >> np.uint64(15))
    x = x * np.uint64(0xBB67AE85) & np.uint64(M32)
    return x ^ (x >> np.uint64(16))


def random_bits(seed, step, tensor, n):
    u = lambda v: np.array([v], dtype=np.uint64)  # noqa: E731
    key = mix(mix(mix(mix(u(seed & M32)) ^ u(seed >> 32)) ^ u(step)) ^ u(tensor))
    return mix(np.arange(n, dtype=np.uint64) ^ key)


def values(code, signed):
    """What a code stands for before its block's scale, from its definition."""
    e, f = (code >> 3 & 15, 10) if signed else (code >> 3, 34)
    v = np.where(e > 0, (8.0 + (code & 7)) * 2.0 ** (np.maximum(e, 1) - f), (code & 7) * 2.0 ** (1 - f))
    return np.where(signed & (code >= 128), -v, v) if signed else v


def held(opt):
    """m and the root of v of each tensor in 64 bits."""
    s = {k: v.cpu() for k, v in opt.state_dict().items()}
    if opt.state_bits == 32:
        return [x.double().numpy() for x in parts(opt, s["exp_avg"])], [x.double().sqrt().numpy() for x in parts(opt, s["exp_avg_sq"])]
    es, er = (s[k].long().numpy().repeat(256) for k in ("exp_avg_scale", "exp_avg_root_scale"))
    m = values(s["exp_avg"].view(torch.uint8).long().numpy(), True) * 2.0 ** (es - 134.0)
    r = values(s["exp_avg_root"].long().numpy(), False) * 2.0 ** (er - 126.0)
    return parts(opt, m), parts(opt, r)


@pytest.mark.parametrize("copies", [True, False])
@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps(bits, offset, grads, copies):
    """Each step from the states as they were held before it: parameters and states within the roundings of one step."""
    opt = make(SIZES, bits, grads, copies, offset=offset)
    (b1, b2), lr, eps, wd = NUMBERS["betas"], NUMBERS["lr"], NUMBERS["eps"], NUMBERS["weight_decay"]
    seed = 1234567890123
    for t in range(1, 5):
        m0, r0 = held(opt)
        v0 = [x.double().cpu().numpy() for x in parts(opt, opt.state_dict()["exp_avg_sq"])] if bits == 32 else [r * r for r in r0]
        w0 = [p.double().cpu().numpy() for p in opt.params]
        opt.step()
        grad = [g.double().cpu().numpy() for g in opt.grads]
        for g in opt.grads:
            g.neg_().mul_(0.5 if t % 2 else 3.0)
        m1, r1 = held(opt)
        for i in range(len(SIZES)):
            g = grad[i]
            # the numbers b1, 1 - b1, .. are rounded to f32 (half a step each), then each operation is
            m, size_m = b1 * m0[i] + (1 - b1) * g, b1 * abs(m0[i]) + (1 - b1) * abs(g)
            v = b2 * v0[i] + (1 - b2) * g * g
            err_m, err_v = 4 * E * size_m + 1e-44, 6 * E * v + 1e-44
            root = np.sqrt(v)
            err_root = 4 * E * root + 1e-23
            denom = root / np.sqrt(1 - b2 ** t) + eps
            by = lr / (1 - b1 ** t)
            w = w0[i] * (1 - lr * wd) - by * m / denom
            err_w = 4 * E * abs(w0[i]) + by / denom * err_m + 10 * E * by * size_m / denom + by * abs(m) / denom ** 2 * err_root / np.sqrt(1 - b2 ** t)
            got = opt.params[i].double().cpu().numpy()
            assert (abs(got - w) <= err_w * 1.01).all(), (t, i)
            if copies:
                assert torch.equal(opt.copies[i], opt.params[i].to(torch.bfloat16))
            if bits == 32:
                assert (abs(m1[i] - m) <= err_m).all() and (abs(r1[i] ** 2 - v) <= err_v + 1e-15 * v).all()
                continue
            rnd = random_bits(seed, t, i, SIZES[i])
            for got, want, err, up, top in ((m1[i], m, err_m, (rnd >> np.uint64(16)).astype(float), 8), (r1[i], root, err_root, (rnd & np.uint64(0xFFFF)).astype(float), 0)):
                for b in range(0, SIZES[i], 256):
                    x, y, u = abs(want[b:b + 256]), abs(got[b:b + 256]), up[b:b + 256]
                    if not x.max():
                        assert not y.any()
                        continue
                    e = max(np.floor(np.log2(x.max() * (1 - 2 * E))), -97)
                    # a step between codes at x: an eighth of its binade, the least binade 14 (m) or 30 (root) below the largest's
                    gap = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(x, 1e-300))), e - (13 if top else 29)) - 3)
                    low = np.floor(x / gap) * gap
                    # the random bits decide but for what f32 is off, and the 2^-16 that 16 bits do not resolve
                    frac, slack = (x - low) / gap, (err[b:b + 256] / gap + 2.0 ** -15) * 1.01
                    goes = u / 65536 + frac
                    ok = np.where(goes > 1 + slack, abs(y - low - gap) <= 1e-12 * y, np.where(goes < 1 - slack, abs(y - low) <= 1e-12 * x, abs(y - x) <= gap * (1 + slack)))
                    # next to a binade's end the steps on its two sides differ
                    edge = abs(np.log2(np.maximum(x, 1e-300)) - np.round(np.log2(np.maximum(x, 1e-300)))) < 1e-6
                    ok |= edge & (abs(y - x) <= 2 * gap)
                    if abs(np.log2(x.max()) - np.round(np.log2(x.max()))) < 1e-6:
                        ok |= abs(y - x) <= 2 * gap
                    assert ok.all(), (t, i, b, top, x[~ok][:3], y[~ok][:3], low[~ok][:3], gap[~ok][:3], goes[~ok][:3])
                    assert (np.sign(got[b:b + 256]) * np.sign(want[b:b + 256]) >= 0).all()
        if bits == 8:
            m, root = opt.state_values()
            for got, want in ((m, m1), (root, r1)):
                assert all(np.array_equal(a.double().cpu().numpy(), b) for a, b in zip(parts(opt, got), want))
    assert opt.state_dict()["steps"].tolist() == [4] * len(SIZES)


def test_rounding_has_no_bias():
    """Over many steps from one state the mean of what is held comes to the exact value: it moves by far less than a code."""
    from randomprojection_amd.optim import AdamW

    n, steps = 4096, 400
    g = torch.Generator(device="cuda").manual_seed(5)
    grad = torch.randn(n, device="cuda", generator=g)
    m, r = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
    for k in range(steps):
        opt = AdamW([torch.zeros(n, device="cuda")], [grad], state_bits=8, seed=k, lr=0.0)
        opt.step()
        a, b = opt.state_values()
        m += a
        r += b
    want_m, want_r = grad.double() * 0.1, (grad.double() ** 2 * 0.001).sqrt()
    for got, want in ((m / steps, want_m), (r / steps, want_r)):
        # a code is off by at most an eighth of the value (where it is not subnormal), so a mean of N by an eighth / (2 sqrt N) in
        # standard deviation at most; over 4096 elements and both states 6 of these bound the largest
        off = (got - want).abs() - want.abs() * (0.125 / 2 / steps ** 0.5 * 6)
        tiny = float(want.abs().max()) * 2.0 ** -14
        assert bool((off <= tiny).all())
        assert abs(float(((got - want) / (want.abs() + tiny)).mean())) < 0.125 / 2 / (steps * n) ** 0.5 * 6


def test_second_moment_falls():
    """With b2 = 0.999 a held v must fall after its gradient has: rounded to the nearest code it never would."""
    from randomprojection_amd.optim import AdamW

    n = 8192
    grad = torch.ones(n, device="cuda")
    opt = AdamW([torch.zeros(n, device="cuda")], [grad], state_bits=8, lr=0.0)
    opt.step()
    grad.zero_()
    for _ in range(1000):
        opt.step()
    mean = float((opt.state_values()[1].double() ** 2).mean())
    # E[root'^2] = v b2 + the variance of the rounding (at most (gap/2)^2 of a step, gap <= root / 8: 1/256 of v, and only as often as the root's
    # change needs a jump: 0.0005 of root a step is at most 0.008 of a gap, so a variance of at most 0.008 gap^2 = 0.000125 v): v falls by
    # 0.000875 to 0.001 a step in the mean
    assert 0.001 * np.exp(-1.05) * 0.97 < mean < 0.001 * np.exp(-0.875) * 1.03


@pytest.mark.parametrize("bits", [32, 8])
def test_active_tensors(bits):
    """A tensor that is not active keeps everything; the others do as they would alone, each with its own step count."""
    opt, alone = make(SIZES, bits), make(SIZES, bits)
    on = torch.tensor([i % 3 != 1 for i in range(len(SIZES))], device="cuda")
    opt.step()
    alone.step()
    before = [p.clone() for p in opt.params], [c.clone() for c in opt.copies], [x.clone() for x in opt.state_dict().values()]
    opt.step(on)
    alone.step()
    steps = opt.state_dict()["steps"].tolist()
    now, then = opt.state_dict(), dict(zip(opt.state_dict(), before[2]))
    for i in range(len(SIZES)):
        assert steps[i] == (2 if on[i] else 1)
        assert torch.equal(opt.params[i], alone.params[i] if on[i] else before[0][i])
        assert torch.equal(opt.copies[i], alone.copies[i] if on[i] else before[1][i])
        for k in ("exp_avg", "exp_avg_sq" if bits == 32 else "exp_avg_root"):
            view = lambda t: t.view(torch.uint8) if bits == 8 else t  # noqa: E731
            assert torch.equal(parts(opt, view(now[k]))[i], parts(opt, view((alone.state_dict() if on[i] else then)[k]))[i])
    opt.step(torch.zeros(len(SIZES), dtype=torch.uint8, device="cuda"))
    assert opt.state_dict()["steps"].tolist() == steps


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits):
    """A gradient that is not finite makes its element NaN, with 8 bits its block's states; other blocks keep their bits."""
    for value in (float("nan"), float("inf"), 3e38):
        opt, clean = make([1000, 600], bits), make([1000, 600], bits)
        opt.grads[0][300] = value
        opt.step()
        clean.step()
        grads = [g.clone() for g in clean.grads]
        for o in (opt, clean):
            for g, h in zip(o.grads, grads):
                g.copy_(h)
            o.step()
        other = torch.ones(1000, dtype=torch.bool, device="cuda")
        if bits == 32:
            other[300] = False
        else:
            other[256:512] = False
            assert torch.isnan(opt.params[0][256:512]).all()
            assert all(torch.isnan(s[256:512]).all() for s in opt.state_values()[1:])
        assert torch.equal(opt.params[0][other], clean.params[0][other]) and torch.equal(opt.params[1], clean.params[1])
        assert all(torch.equal(a, b) for a, b in zip(parts(opt, opt.state_values()[0])[1:], parts(clean, clean.state_values()[0])[1:]))


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_and_huge(bits):
    """Values far from 1: scales at both ends of their range."""
    from randomprojection_amd.optim import AdamW

    for by in (1e-38, 1e-30, 1e-20, 1e10, 1e18):
        g = (torch.randn(512, generator=torch.Generator().manual_seed(1)) * by).cuda()
        opt = AdamW([torch.zeros(512, device="cuda")], [g], state_bits=bits, eps=0.0 if by > 1e-18 else 1e-8, lr=1e-3, weight_decay=0.0)
        opt.step()
        m, root = opt.state_values()
        want = (g.double() * 0.1)
        assert torch.isfinite(opt.params[0]).all() and torch.isfinite(m).all() and torch.isfinite(root).all()
        # 8 bits: a step between codes is at most an eighth; the least scale is 2^-97, of which the least code is 2^-16 (m: 2^-113 = 1e-34)
        assert bool(((m.double() - want).abs() <= want.abs() * 0.13 + (1e-34 if bits == 8 else 1e-44) + float(want.abs().max()) * 2.0 ** -15).all())
        if by > 1e-18:
            # the first step goes by lr, whatever the gradient's size
            assert bool(((opt.params[0].double().abs() - 1e-3).abs() <= 1e-3 * 1e-5).all())


def test_load_state_other_stream_and_graph():
    """States carried over continue bit for bit; another stream and a replayed graph do what eager steps do."""
    for bits in (32, 8):
        a, b, c = make(SIZES, bits), make(SIZES, bits), make(SIZES, bits)
        for _ in range(3):
            a.step()
            b.step()
        fresh = make(SIZES, bits)
        fresh.load_state_dict(b.state_dict())
        for p, q in zip(fresh.params, b.params):
            p.copy_(q)
        with pytest.raises(ValueError, match="states held"):
            fresh.load_state_dict({"steps": a.state_dict()["steps"]})
        with pytest.raises(ValueError, match="steps must be"):
            fresh.load_state_dict(a.state_dict() | {"steps": a.state_dict()["steps"][:-1]})
        with pytest.raises(ValueError, match="active"):
            a.step(torch.ones(3, device="cuda", dtype=torch.uint8))
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        c.step()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            c.step()
        for _ in range(3):  # the capture itself did nothing
            g.replay()
            a.state_values()
            torch.cuda.synchronize()
        a.step()
        fresh.step(stream=side.cuda_stream)
        side.synchronize()
        for x in (fresh, c):
            assert all(torch.equal(p, q) for p, q in zip(x.params + x.copies, a.params + a.copies))
            for k, v in a.state_dict().items():
                u = x.state_dict()[k]
                assert torch.equal(u.view(torch.uint8), v.view(torch.uint8)), k


def test_projection_gradient_and_step_together():
    """A few training steps of adapters as they are used: the projection reads the copies, the gradients go where the optimizer reads
    them, eager and as one graph; each step's outputs against 64 bits."""
    from randomprojection_amd.adapters import adapted_project_backward_device, adapted_project_device, prepare_bank
    from randomprojection_amd.optim import AdamW

    n, m, p, G, R = 200, 256, 128, 5, 8
    rand = torch.Generator(device="cuda").manual_seed(3)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=rand)  # noqa: E731
    X, C = normal(n, m).bfloat16(), (normal(p, m) * p ** -0.5).bfloat16()
    ids = torch.randint(-1, G, (n,), device="cuda", generator=rand, dtype=torch.int32)
    target = normal(n, p)

    class Model:
        def __init__(self, bits):
            r = torch.Generator(device="cuda").manual_seed(4)
            self.down, self.up = torch.randn(G, R, m, device="cuda", generator=r) * m ** -0.5, torch.zeros(G, R, p, device="cuda")
            self.low = self.down.bfloat16(), self.up.bfloat16()
            self.grad = torch.zeros_like(self.down), torch.zeros_like(self.up)
            per = lambda ts: [t[g] for t in ts for g in range(G)]  # noqa: E731
            self.opt = AdamW(per((self.down, self.up)), per(self.grad), lr=1e-2, copies=per(self.low), state_bits=bits, seed=9)
            self.C, self.Ct = prepare_bank(C, "bf16"), prepare_bank(C.T, "bf16")

        def step(self):
            kw = dict(compute="bf16", prepared=True)
            Y, h = adapted_project_device(X, self.C, *self.low, ids, return_hidden=True, **kw)
            dY = (Y - target).bfloat16()
            dX, _, _ = adapted_project_backward_device(dY, X, self.Ct, *self.low, ids, h, out=self.grad, **kw)
            self.opt.step()
            return Y, dY, dX

    for bits in (32, 8):
        eager, captured = Model(bits), Model(bits)
        got = [eager.step()]
        captured.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = captured.step()
        for k in range(4):
            got = eager.step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, out))
            assert torch.equal(eager.down, captured.down) and torch.equal(eager.up, captured.up)
            assert torch.equal(eager.low[0], eager.down.bfloat16()) and torch.equal(eager.low[1], eager.up.bfloat16())
        down, up = (t.double() for t in eager.low)
        Y, h = adapted_project_device(X, eager.C, *eager.low, ids, return_hidden=True, compute="bf16", prepared=True)
        want = X.double() @ C.double().T
        size = X.double().abs() @ C.double().abs().T
        for g in range(G):
            at = torch.nonzero(ids == g)[:, 0]
            want[at] += X[at].double() @ down[g].T @ up[g]
            size[at] += X[at].double().abs() @ down[g].T.abs() @ up[g].abs()
        assert bool(((Y.double() - want).abs() <= (m + R + 8) * 2.0 ** -23 * size).all())


@pytest.mark.parametrize("grads", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("more", [[768 * 256 - 321 * 256], [768 * 256 - 321 * 256 + 1], [9000 * 256 + 5], [1] * 244, [1] * 245, [0] * 600])
def test_longer_lists_step_alike(more, bits, grads):
    """The first tensors of a list get the same bits whatever follows them, whichever form of the step its length takes; eagerly, with
    tensors left out, and from a graph."""
    short, long = make(SIZES, bits, grads), make(SIZES + more, bits, grads)
    T = len(SIZES)
    for a, b in zip(long.params[:T] + long.grads[:T], short.params + short.grads):  # drawn after all parameters, the gradients differ
        a.copy_(b)
    assert sum(-(-s // 256) for s in SIZES) == 321
    some = torch.tensor([i % 3 != 1 for i in range(T)] + [i % 2 == 0 for i in range(len(more))], device="cuda")
    graphs = []
    for opt in (short, long):
        active = some[:len(opt.params)].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
            opt.step(active)
        graphs.append((opt, graph, active))
    for k in range(3):
        for opt, graph, active in graphs:
            opt.step()
            opt.step(active)
            for _ in range(2):
                graph.replay()
            for g in opt.grads:
                g.mul_(-0.5)
    torch.cuda.synchronize()
    for a, b in zip(short.params + short.copies, long.params[:T] + long.copies[:T]):
        assert torch.equal(a, b)
    for x, y in zip(held(short), held(long)):
        assert all(np.array_equal(a, b) for a, b in zip(x, y))
    want = [18 if s else 9 for s in some.tolist()]
    assert long.state_dict()["steps"].tolist() == want and short.state_dict()["steps"].tolist() == want[:T]
