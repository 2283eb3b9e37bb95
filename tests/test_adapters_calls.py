"""Adapters beside the dense projection and AdamW: which stream a call takes, sizes at the limits, checked without a GPU."""
import contextlib
import ctypes

import pytest
import torch

from randomprojection_amd import _native as nat
from randomprojection_amd import adapters, optim


class _Stream:
    def __init__(self, handle):
        self.cuda_stream, self.device, self.waited = handle, torch.device("cuda", 0), []

    def wait_stream(self, other):
        self.waited.append(other)


@pytest.fixture
def streams(monkeypatch):
    """torch's streams as they are where the current one is a side stream: handle 0 is the default stream, and an
    ExternalStream of 0 would be a stream of its own."""
    made = {0: _Stream(0), 111: _Stream(111)}
    external = lambda handle, device=None: made.setdefault(handle or 999, _Stream(handle or 999))  # noqa: E731
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: made[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: made[111])
    monkeypatch.setattr(torch.cuda, "ExternalStream", external)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext(s))
    for module in (adapters, optim):
        monkeypatch.setattr(module, "raw_stream", lambda device: 111)
    return made


@pytest.mark.parametrize("handle", [0, 222, 111, None])
def test_the_stream_that_is_named_waits_for_the_current_one(streams, handle):
    """The default stream's handle is 0: it is that stream that has to wait for the casts queued on the current one."""
    class Temporary:
        kept = []

        def record_stream(self, s):
            self.kept.append(s)

    dev = torch.device("cuda", 0)
    opt = optim.AdamW.__new__(optim.AdamW)
    opt.device = dev
    for call in (lambda t: adapters._on_stream(handle, dev, (t, None)), lambda t: opt._stream(handle, t, None)):
        temporary = Temporary()
        temporary.kept = []
        for s in streams.values():
            s.waited.clear()
        assert call(temporary) == (111 if handle is None else handle)
        other = handle not in (None, 111)
        assert temporary.kept == ([streams[handle]] if other else [])
        assert {k: v.waited for k, v in streams.items() if v.waited} == ({handle: [streams[111]]} if other else {})


def test_state_values_take_the_stream_in_both_widths(streams):
    """States in 32 bits are read out on the stream that is named too, behind the steps queued there."""
    opt = optim.AdamW.__new__(optim.AdamW)
    opt.device, opt.state_bits = torch.device("cpu"), 32
    opt.state = {"exp_avg": torch.tensor([1.0, -2.0]), "exp_avg_sq": torch.tensor([9.0, 0.25])}
    entered, current = [], torch.cuda.stream
    torch.cuda.stream = lambda s: entered.append(s) or current(s)  # the fixture puts torch's own back
    torch.Tensor.record_stream, record = lambda t, s: None, torch.Tensor.record_stream
    try:
        for handle, waits in ((None, []), (111, []), (0, [streams[111]]), (222, [streams[111]])):
            entered.clear()
            m, root = opt.state_values(stream=handle)
            assert torch.equal(m, opt.state["exp_avg"]) and torch.equal(root, torch.tensor([3.0, 0.5]))
            assert m.data_ptr() != opt.state["exp_avg"].data_ptr()
            if waits:
                assert entered == [streams[handle]] and streams[handle].waited == waits
            else:
                assert entered in ([], [None])
    finally:
        torch.Tensor.record_stream = record


def test_seed_is_as_fitted(monkeypatch):
    """What the optimizer rounds by is the seed of the last fit, whenever it is made and whatever was set since; it travels in a pickle."""
    import pickle

    import numpy as np

    from randomprojection_amd import AdaptedGaussianProjection, gaussian

    made = []

    class Optimizer:
        def __init__(self, params, grads, *, seed, **kw):
            made.append(seed)

    device = torch.device
    monkeypatch.setattr(torch, "device", lambda *a: device("cpu"))
    monkeypatch.setattr(optim, "AdamW", Optimizer)
    monkeypatch.setattr(gaussian, "_torch", lambda: torch)
    X = np.random.default_rng(0).standard_normal((20, 33))
    est = AdaptedGaussianProjection(n_components=7, n_adapters=3, rank=2, random_state=5, seed=4).fit(X)
    est.set_params(seed=9)
    pickle.loads(pickle.dumps(est))._on_device()
    est._on_device()
    est.set_params(seed=9).fit(X)._on_device()
    assert made == [4, 4, 9]


@pytest.mark.parametrize("dtype", [nat.RP_F32, nat.RP_BF16])
def test_workspace_without_rows_holds_the_counts(dtype):
    """Over 700 adapters the gradients of an empty batch count its rows as those of a longer one do: five lists of an entry an adapter and 16
    bytes of each one's chunk."""
    for G in (701, 4000, 16383):
        for what in (nat.RP_ADAPT_GRADIENTS, nat.RP_ADAPT_GRADIENTS_DX):
            assert nat.load().rp_adapt_workspace_bytes(dtype, 0, 70, 20, G, 1, what) >= (5 * 4 + 16) * G


def test_calls_whose_grids_would_not_fit_are_refused():
    """An axis of a grid has fewer than 2^32 threads: sizes past that are refused before anything is launched, those below are not."""
    lib = nat.load()
    size = lambda dtype, what, **kw: lib.rp_adapt_workspace_bytes(  # noqa: E731
        dtype, *(({"n": 1, "m": 64, "p": 1, "G": 1, "R": 1} | kw).values()), what)
    project, banks, both = nat.RP_ADAPT_PROJECT, nat.RP_ADAPT_GRADIENTS, nat.RP_ADAPT_GRADIENTS_DX
    most = 2 ** 31 - 513
    for dtype, what, over, under in (
            (nat.RP_F32, project, {"m": most}, {"m": most - 8192}),  # few rows: 2^23 blocks of 512 threads, 8 lines of 32 columns each
            (nat.RP_F32, both, {"p": most}, {"p": most - 8192}),
            (nat.RP_BF16, project, {"n": 2 ** 31 - 1, "p": 64}, {"n": 2 ** 30 - 4096, "p": 64}),  # 64 rows a block of the shrink
            (nat.RP_BF16, banks, {"n": 2 ** 31 - 1}, {"n": 2 ** 30 - 4096}),
            (nat.RP_BF16, banks, {"G": 16383, "m": 2 ** 24 + 2048}, {"G": 16383, "m": 65536}),  # 2^31 blocks of outer products
            (nat.RP_F32, both, {"G": 16383, "m": 2 ** 23 + 2048}, {"G": 16383, "m": 65536, "p": 64})):
        assert size(dtype, what, **under) > 0 and size(dtype, what, **over) == -1, (what, over, under)
        assert b"one launch" in lib.rp_last_error()
    a = 1 << 20  # never read
    assert lib.rp_adapt_project_device(0, a, most + 1, nat.RP_F32, 1, most, a, 1, a, a, 1, 1, None, a, a, 1, None, a, 1 << 40, None) == nat.RP_ERR_UNSUPPORTED
    assert lib.rp_adapt_gradients_device(0, a, 64, a, 2 ** 25, nat.RP_BF16, 1, 2 ** 24 + 2048, 1, None, a, a, 16383, 1, None, a, a, None, 0, a, 2 ** 25, 2 ** 25,
                                         a, 1, 1, a, 1 << 50, None) == nat.RP_ERR_UNSUPPORTED


def test_adamw_refuses_lists_whose_grid_would_not_fit():
    """2^26 waves of 64 threads, a wave for 1024 elements: refused from the sizes alone, before any table is made."""
    lib, a, h = nat.load(), 1 << 20, ctypes.c_void_p()
    for sizes in ([2 ** 36], [2 ** 38], [2 ** 35, 2 ** 35, 1]):
        T = len(sizes)
        many = (ctypes.c_void_p * T)(*[a] * T)
        rc = lib.rp_adamw_create(0, T, (ctypes.c_int64 * T)(*sizes), many, many, nat.RP_F32, None, 32, a, a, None, None, a, ctypes.byref(h))
        assert rc == nat.RP_ERR_UNSUPPORTED and b"too many elements" in lib.rp_last_error() and not h


def test_a_state_without_the_seed_of_its_fit_takes_the_one_it_has():
    import numpy as np

    from randomprojection_amd import AdaptedGaussianProjection

    est = AdaptedGaussianProjection(n_components=7, n_adapters=3, rank=2, random_state=5, seed=4)
    again = AdaptedGaussianProjection()
    again.__setstate__(est.__getstate__())  # not fitted
    assert not hasattr(again, "_seed")
    state = est.fit(np.random.default_rng(0).standard_normal((20, 33))).__getstate__()
    for state, seed in ((state, 4), ({k: v for k, v in state.items() if k != "_seed"} | {"seed": 6}, 6)):
        again.__setstate__(state)
        assert again._seed == seed


def test_workspace_of_no_such_call_is_refused():
    lib = nat.load()
    for what in (-1, 3, 7):
        for n in (0, 3, 1000):
            assert lib.rp_adapt_workspace_bytes(nat.RP_BF16, n, 100, 50, 4, 8, what) == -1 and b"what" in lib.rp_last_error()


def test_loads_to_lds_wait_for_their_destination():
    """A load to LDS takes its destination from M0 and needs one instruction between it and the write of M0; the compiler puts it there, inline
    asm has to."""
    import pathlib
    import re

    import randomprojection_amd

    found = 0
    for source in sorted((pathlib.Path(randomprojection_amd.__file__).parent / "csrc").glob("*.hip")):
        for text in re.findall(r'asm volatile\(((?:\s*"(?:[^"\\]|\\.)*")+)', source.read_text()):
            steps = [s.strip() for s in re.sub(r'"\s*"', "", text).strip().strip('"').replace("\\t", "").split("\\n")]
            for i, s in enumerate(steps):
                if "load_lds" in s or ("buffer_load" in s and s.endswith("lds")):
                    found += 1
                    writes = [k for k in range(i) if " m0," in steps[k]]
                    assert writes and i - writes[-1] >= 2, (source.name, steps)
    assert found
