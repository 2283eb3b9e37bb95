"""Cases of the adapted dense projection, its gradients and the AdamW step, for timing and comparing.

``run`` computes a case in its plain form (elementary torch operations in 32 bits), or, where ``own`` is
true, by the calls a user makes of the package. Symbols: n rows of m features, a shared projection of p
components, G adapters of rank r; row i has the adapter ids[i], or none where that is -1."""
import torch

own = False

STEP = {"bf16": 64, "fp32": 32}  # the contraction's width is padded to a multiple of this, as for the shared projection
TYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 256  # elements that share one scale of a state in 8 bits
M32 = 0xFFFFFFFF


def listed():
    f, g, a = "project", "gradients", "adamw"
    return [
        # one request's single row: latency
        {"name": "project-one-row", "op": f, "type": "bf16", "n": 1, "m": 4096, "p": 1024, "G": 8, "r": 16, "rows": "single", "hidden": False},
        # single rows of 64 requests, an adapter of its own nearly each: reads C and the adapters once
        {"name": "project-single-rows", "op": f, "type": "bf16", "n": 64, "m": 16384, "p": 1024, "G": 64, "r": 16, "rows": "single", "hidden": False},
        # requests of many rows packed together, a larger rank
        {"name": "project-requests", "op": f, "type": "bf16", "n": 1777, "m": 4096, "p": 4096, "G": 24, "r": 64, "rows": "packed", "hidden": False},
        # the dense configuration's width, one block of rows as the estimator streams them
        {"name": "project-bulk", "op": f, "type": "bf16", "n": 65536, "m": 16384, "p": 1024, "G": 32, "r": 16, "rows": "packed", "hidden": True},
        # exact products, odd sizes
        {"name": "project-fp32-odd", "op": f, "type": "fp32", "n": 1003, "m": 4001, "p": 200, "G": 5, "r": 7, "rows": "packed", "hidden": True},
        # a small training batch on fixed features (no gradient of the rows)
        {"name": "gradients-small", "op": g, "type": "bf16", "n": 300, "m": 4096, "p": 200, "G": 4, "r": 8, "rows": "packed", "dx": False},
        # a training batch of the dense configuration's width, with the rows' gradient
        {"name": "gradients-wide", "op": g, "type": "bf16", "n": 16384, "m": 16384, "p": 1024, "G": 16, "r": 16, "rows": "packed", "dx": True},
        # exact products, odd sizes, rows of every adapter in turn
        {"name": "gradients-fp32-odd", "op": g, "type": "fp32", "n": 2049, "m": 1000, "p": 129, "G": 6, "r": 5, "rows": "single", "dx": True},
        # a few small adapters: latency
        {"name": "adamw-few", "op": a, "bits": 32, "tensors": 16, "sizes": "ragged", "least": 100, "most": 20000, "grads": "fp32", "copies": True},
        # 256 adapters of the dense configuration (down 16 x 16384, up 16 x 1024) with their bf16 operands
        {"name": "adamw-bank", "op": a, "bits": 32, "tensors": 512, "sizes": "pairs", "least": 16384, "most": 262144, "grads": "fp32", "copies": True},
        # the same with states in 8 bits
        {"name": "adamw-bank-8bit", "op": a, "bits": 8, "tensors": 512, "sizes": "pairs", "least": 16384, "most": 262144, "grads": "fp32", "copies": True},
        # many tensors of ragged sizes, gradients in bf16
        {"name": "adamw-ragged-8bit", "op": a, "bits": 8, "tensors": 300, "sizes": "ragged", "least": 1, "most": 100000, "grads": "bf16", "copies": False},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(["project", "project", "gradients", "adamw"])
    if op == "adamw":
        most = log(100, 262144)
        return {"op": op, "bits": rng.choice([8, 32]), "tensors": log(1, 512), "sizes": rng.choice(["pairs", "ragged"]), "least": log(1, most), "most": most,
                "grads": rng.choice(["fp32", "bf16"]), "copies": rng.random() < 0.5}
    kind = rng.choice(["bf16", "bf16", "fp32"])
    n, m, p = log(1, 65536), log(64, 16384), log(16, 4096)
    most = 2.2e12 if kind == "bf16" and op == "project" else 5e11  # no more products than the largest listed case has
    while 2 * n * m * p > most:
        n = n // 2
    case = {"op": op, "type": kind, "n": n, "m": m, "p": p, "G": log(1, 64), "r": log(1, 64), "rows": rng.choice(["packed", "single"])}
    if op == "project":
        case["hidden"] = rng.random() < 0.5
    else:
        case["dx"] = rng.random() < 0.5
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _padded(t, step):
    return torch.nn.functional.pad(t, (0, -t.shape[-1] % step)).contiguous()


def _sizes(case):
    """Elements of each tensor: the two kinds of an adapter in turn, or spread over their logarithm."""
    T, least, most = case["tensors"], case["least"], case["most"]
    if case["sizes"] == "pairs":
        return [most if t % 2 == 0 else least for t in range(T)]
    spread = torch.rand(T, generator=torch.Generator().manual_seed(0)).tolist()
    return [min(most, max(least, round(least * (most / least) ** x))) for x in spread]


def _ids(case, seed):
    """The adapter of each row: of single rows at random, of requests of about a hundred rows in runs; about one request in ten has none."""
    g = torch.Generator().manual_seed(seed)
    n = case["n"]
    pick = torch.randint(0, case["G"], (n,), generator=g)
    pick[torch.rand(n, generator=g) < 0.1] = -1
    if case["rows"] == "packed":
        request = torch.cumsum((torch.rand(n, generator=g) < 0.01).to(torch.int64), 0)
        pick = pick[request]
    return pick.to(torch.int32).cuda()


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["op"] == "adamw":
        return _prepare_adamw(state, seed, g)
    n, m, p, G, r = (case[k] for k in ("n", "m", "p", "G", "r"))
    kind, step = TYPE[case["type"]], STEP[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * by).to(kind)

    state["X"] = normal(n, m)
    C = normal(p, m, by=p ** -0.5)  # a Gaussian projection's components
    state["C"] = _padded(C, step)
    state["down"] = _padded(normal(G, r, m, by=m ** -0.5), step)
    state["up"] = _padded(normal(G, r, p, by=r ** -0.5), step)
    state["scale"] = torch.rand(G, device="cuda", generator=g) * 1.5 + 0.5
    state["ids"] = _ids(case, seed)
    if case["op"] == "gradients":
        state["dY"] = normal(n, p, by=1 / n)
        if case["dx"]:
            state["Ct"] = _padded(C.T, step)
        has = (state["ids"].long()[:, None] == torch.arange(G, device="cuda")).float()
        every = (state["X"].float() @ state["down"][..., :m].float().reshape(G * r, m).T).reshape(n, G, r)
        state["hidden"] = (every * has[:, :, None]).sum(1)  # what the forward pass kept
    return state


def _prepare_adamw(state, seed, g):
    """Parameters and gradients of all tensors in one buffer each, a tensor at a multiple of BLOCK; the states as they stand after some steps."""
    T, sizes = state["tensors"], _sizes(state)
    blocks = [-(-s // BLOCK) for s in sizes]
    state["sizes"], state["offsets"] = sizes, [0]
    for b in blocks:
        state["offsets"].append(state["offsets"][-1] + b * BLOCK)
    nb = sum(blocks)
    of = torch.repeat_interleave(torch.arange(T), torch.tensor(blocks)).cuda()
    state["of"] = of  # the tensor of each block
    state["first"] = torch.tensor(state["offsets"][:-1]).cuda()
    at = torch.arange(nb, device="cuda")[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") - state["first"][of][:, None]
    state["valid"] = at < torch.tensor(sizes).cuda()[of][:, None]
    live = state["valid"].float()

    def normal(by):
        return torch.randn(nb, BLOCK, device="cuda", generator=g) * by * live

    # gradients whose size varies from tensor to tensor, as those of adapters with more and fewer rows do
    size = torch.exp(torch.randn(T, device="cuda", generator=g) - 7)[of][:, None]
    state["params"] = normal(0.02)
    state["grads"] = (normal(1.0) * size).to(TYPE[state["grads"]])
    m = normal(0.3) * size
    v = (torch.rand(nb, BLOCK, device="cuda", generator=g) + 0.01) * live * size * size
    state["steps"] = torch.randint(1, 2000, (T,), generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    if state["bits"] == 32:
        state["m"], state["v"] = m, v
    else:  # to the nearest code
        state["m_scale"], root = _exponent(m), v.sqrt()
        state["v_scale"] = _exponent(root)
        t = (m.abs() * _power(134 - state["m_scale"]) * 2.0 ** -120).contiguous().view(torch.int32)
        state["m"] = ((t + 0x80000 >> 20) | (m < 0).int() * 128).to(torch.uint8).view(torch.float8_e4m3fn)
        t = (root * _power(126 - state["v_scale"]) * 2.0 ** -96).contiguous().view(torch.int32)
        state["v"] = (t + 0x80000 >> 20).to(torch.uint8)
    state["copy"] = torch.zeros(nb, BLOCK, device="cuda", dtype=torch.bfloat16) if state["copies"] else None
    state |= {"lr": 1e-3, "b1": 0.9, "b2": 0.999, "eps": 1e-8, "decay": 0.01, "seed": seed * 7919 + 1}
    if own:  # the optimizer that a program keeps: over the same buffers, tensor by tensor
        from randomprojection_amd.optim import AdamW

        def views(flat):
            return [flat.view(-1)[o:o + s] for o, s in zip(state["offsets"], sizes)]

        opt = AdamW(views(state["params"]), views(state["grads"]), lr=state["lr"], betas=(state["b1"], state["b2"]), eps=state["eps"], weight_decay=state["decay"],
                    state_bits=state["bits"], copies=None if state["copy"] is None else views(state["copy"]), seed=state["seed"])
        kept = {"steps": state["steps"], "exp_avg": state["m"].view(-1), "exp_avg_sq" if state["bits"] == 32 else "exp_avg_root": state["v"].view(-1)}
        if state["bits"] == 8:
            kept |= {"exp_avg_scale": state["m_scale"].view(-1).to(torch.uint8), "exp_avg_root_scale": state["v_scale"].view(-1).to(torch.uint8)}
        opt.load_state_dict(kept)
        state["opt"] = opt
    return state


def run(state):
    if state["op"] == "project":
        return _project(state)
    return _gradients(state) if state["op"] == "gradients" else _adamw(state)


def _project(s):
    if own:
        from randomprojection_amd.adapters import adapted_project_device

        got = adapted_project_device(s["X"], s["C"], s["down"], s["up"], s["ids"], scale=s["scale"], compute=s["type"], prepared=True, return_hidden=s["hidden"])
        return {"Y": got[0], "hidden": got[1]} if s["hidden"] else {"Y": got}
    n, m, p, G, r = (s[k] for k in ("n", "m", "p", "G", "r"))
    X = s["X"].float()
    has = (s["ids"].long()[:, None] == torch.arange(G, device="cuda"))[:, :, None]
    every = (X @ s["down"][..., :m].float().reshape(G * r, m).T).reshape(n, G, r)
    every = torch.where(has, every, 0.0)
    Y = X @ s["C"][:, :m].float().T
    Y = Y + (every * s["scale"][:, None]).reshape(n, G * r) @ s["up"][..., :p].float().reshape(G * r, p)
    return {"Y": Y, "hidden": every.sum(1)} if s["hidden"] else {"Y": Y}


def _gradients(s):
    if own:
        from randomprojection_amd.adapters import adapted_project_backward_device

        got = adapted_project_backward_device(s["dY"], s["X"], s.get("Ct"), s["down"], s["up"], s["ids"], s["hidden"], scale=s["scale"], compute=s["type"], prepared=True)
        return {k: v for k, v in zip(("dX", "d_down", "d_up"), got) if v is not None}
    n, m, p, G, r = (s[k] for k in ("n", "m", "p", "G", "r"))
    X, dY = s["X"].float(), s["dY"].float()
    has = (s["ids"].long()[:, None] == torch.arange(G, device="cuda"))[:, :, None]
    scale = s["scale"][:, None]
    t = torch.where(has, (dY @ s["up"][..., :p].float().reshape(G * r, p).T).reshape(n, G, r) * scale, 0.0).reshape(n, G * r)
    h = torch.where(has, s["hidden"][:, None, :] * scale, 0.0).reshape(n, G * r)
    got = {"d_down": (t.T @ X).reshape(G, r, m), "d_up": (h.T @ dY).reshape(G, r, p)}
    if s["dx"]:
        got["dX"] = (dY @ s["Ct"][:, :p].float().T + t @ s["down"][..., :m].float().reshape(G * r, m)).to(s["X"].dtype)
    return got


def _exponent(x):
    """The biased exponent of each block's largest magnitude, in the range a scale can take."""
    return (x.abs().amax(1, keepdim=True).view(torch.int32) >> 23).clamp(30, 254)


def _power(e):
    """2.0 ** e for whole e within the normal range."""
    return (e + 127 << 23).view(torch.float32)


def _mix(x):
    """32 bits to 32 bits, held in 64."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _values(s):
    """The states in 8 bits as the values they stand for."""
    code = s["m"].view(torch.uint8).int()
    m = ((code & 127) << 20).view(torch.float32) * 2.0 ** 120 * _power(s["m_scale"] - 134)
    m = torch.where(code >= 128, -m, m)
    root = (s["v"].int() << 20).view(torch.float32) * 2.0 ** 96 * _power(s["v_scale"] - 126)
    return m, root


def _adamw(s):
    if own:
        s["opt"].step()
        got = {"params": s["params"]}
        if s["copy"] is not None:
            got["copy"] = s["copy"]
        if s["bits"] == 32:
            kept = s["opt"].state_dict()
            return got | {"m": kept["exp_avg"].view(-1, BLOCK), "v": kept["exp_avg_sq"].view(-1, BLOCK)}
        m, root = s["opt"].state_values()
        return got | {"m": m.view(-1, BLOCK), "root": root.view(-1, BLOCK)}
    of = s["of"]
    s["steps"] += 1
    t = s["steps"].double()
    by = (s["lr"] / (1 - s["b1"] ** t)).float()[of][:, None]
    rs = (1 / (1 - s["b2"] ** t).sqrt()).float()[of][:, None]
    if s["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, root = _values(s)
        v = root * root
    g = s["grads"].float()
    m = m * s["b1"] + g * (1 - s["b1"])
    v = v * s["b2"] + g * g * (1 - s["b2"])
    root = v.sqrt()
    s["params"].copy_(s["params"] * (1 - s["lr"] * s["decay"]) - m / (root * rs + s["eps"]) * by)
    got = {"params": s["params"]}
    if s["copy"] is not None:
        s["copy"].copy_(s["params"])
        got["copy"] = s["copy"]
    if s["bits"] == 32:
        s["m"], s["v"] = m, v
        return got | {"m": m, "v": v}
    seed = s["seed"]
    tensor = torch.arange(s["tensors"], device="cuda")
    key = _mix(_mix(torch.full_like(tensor, seed & M32)) ^ (seed >> 32 & M32))
    key = _mix(_mix(key ^ s["steps"].long()) ^ tensor)
    at = torch.arange(of.numel(), device="cuda")[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") - s["first"][of][:, None]
    bits = _mix(at ^ key[of][:, None])
    s["m_scale"], s["v_scale"] = _exponent(m), _exponent(root)
    code = (m.abs() * _power(134 - s["m_scale"]) * 2.0 ** -120).view(torch.int32) + ((bits >> 16 << 4) + 8).int() >> 20
    s["m"] = (code | (m.view(torch.int32) < 0).int() * 128).to(torch.uint8).view(torch.float8_e4m3fn)
    s["v"] = ((root * _power(126 - s["v_scale"]) * 2.0 ** -96).view(torch.int32) + (((bits & 0xFFFF) << 4) + 8).int() >> 20).to(torch.uint8)
    m, root = _values(s)
    return got | {"m": m, "root": root}


def work(case):
    if case["op"] == "adamw":
        total = sum(_sizes(case))
        each = 8 + (4 if case["grads"] == "fp32" else 2) + (2 if case["copies"] else 0)
        each += 16 if case["bits"] == 32 else 4 + 2 + 8  # in 8 bits: codes read and written, then read and written as values
        return {"bytes": total * each, "flops": total * 15}
    n, m, p, G, r = (case[k] for k in ("n", "m", "p", "G", "r"))
    e = 2 if case["type"] == "bf16" else 4
    used = min(n, G)
    if case["op"] == "project":
        return {"bytes": e * (n * m + p * m + used * r * (m + p)) + 4 * n * p + (4 * n * r if case["hidden"] else 0) + 4 * n,
                "flops": 2 * n * m * p + 2 * n * r * (m + p)}
    bytes_, flops = e * (n * m + n * p + used * r * p) + 4 * n * r + 4 * G * r * (m + p) + 4 * n, 2 * n * r * (2 * p + m)
    if case["dx"]:
        bytes_, flops = bytes_ + e * (n * m + p * m + used * r * m), flops + 2 * n * m * (p + r)
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    m, p, G, r, n = (case[k] for k in ("m", "p", "G", "r", "n"))
    X, down, up, scale = s["X"].double(), s["down"][..., :m].double(), s["up"][..., :p].double(), s["scale"].double()
    ids = s["ids"].long()
    if case["op"] == "project":
        Y, H = X @ s["C"][:, :m].double().T, X.new_zeros(n, r)
        for g in range(G):
            at = torch.nonzero(ids == g)[:, 0]
            H[at] = X[at] @ down[g].T
            Y[at] += scale[g] * (H[at] @ up[g])
        return {"Y": Y, "hidden": H} if case["hidden"] else {"Y": Y}
    dY, H = s["dY"].double(), s["hidden"].double()
    got = {"d_down": X.new_zeros(G, r, m), "d_up": X.new_zeros(G, r, p)}
    if case["dx"]:
        got["dX"] = dY @ s["Ct"][:, :p].double().T
    for g in range(G):
        at = torch.nonzero(ids == g)[:, 0]
        t = scale[g] * (dY[at] @ up[g].T)
        got["d_down"][g] = t.T @ X[at]
        got["d_up"][g] = scale[g] * (H[at].T @ dY[at])
        if case["dx"]:
            got["dX"][at] += t @ down[g]
    return got


def _exact_adamw(s):
    """The parameters; the states where they are held in 32 bits (which code of 8 bits one comes to goes by the last bit of a random rounding)."""
    if s["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        bits = s["m"].view(torch.uint8).long()
        e, f = bits >> 3 & 15, (bits & 7).double()
        m = torch.where(e > 0, (8 + f) * 2.0 ** (e.double() - 10), f * 2.0 ** -9) * torch.where(bits > 127, -1.0, 1.0).double()
        m = m * 2.0 ** (s["m_scale"].double() - 134)
        bits = s["v"].long()
        e, f = bits >> 3, (bits & 7).double()
        v = (torch.where(e > 0, (8 + f) * 2.0 ** (e.double() - 34), f * 2.0 ** -33) * 2.0 ** (s["v_scale"].double() - 126)) ** 2
    g, t = s["grads"].double(), (s["steps"].double() + 1)[s["of"]][:, None]
    m = s["b1"] * m + (1 - s["b1"]) * g
    v = s["b2"] * v + (1 - s["b2"]) * g ** 2
    p = s["params"].double() * (1 - s["lr"] * s["decay"])
    p = p - s["lr"] * (m / (1 - s["b1"] ** t)) / ((v / (1 - s["b2"] ** t)).sqrt() + s["eps"])
    got = {"params": p}
    if s["copy"] is not None:
        got["copy"] = p
    if s["bits"] == 32:
        return got | {"m": m, "v": v}
    return got | {"m": None, "root": None}
