"""A Gaussian projection that many tenants share, with a small learned part for each.

``GaussianRandomProjection`` gives every row the same frozen components. ``AdaptedGaussianProjection`` keeps them and lets each of
``n_adapters`` tenants learn a low-rank correction of its own beside them, from targets for its rows: one call serves and one call trains rows
of any mix of tenants (``adapters.py`` has the products, ``optim.py`` the AdamW step; no reference counterpart).
"""
from __future__ import annotations

import numpy as np
from sklearn.utils import check_array, check_random_state
from sklearn.utils.validation import check_is_fitted, validate_data

from .gaussian import _STEP, GaussianRandomProjection

__all__ = ["AdaptedGaussianProjection"]


class _Bank:
    """The adapters on the device: float32 parameters padded to the kernels' width, their gradients, the operands of the compute type
    (rounded copies in "bf16", the parameters themselves in "fp32") and the optimizer, one tensor for each adapter and kind."""

    def __init__(self, est, components, down, up, state=None):
        import torch

        from .adapters import prepare_bank
        from .optim import AdamW

        dev, mode, G = torch.device("cuda", est.device), est._mode(), down.shape[0]
        self.made_for = est._made_for()
        pad = lambda a: torch.nn.functional.pad(torch.as_tensor(a, device=dev), (0, -a.shape[-1] % _STEP[mode]))  # noqa: E731
        C = torch.as_tensor(np.ascontiguousarray(components, dtype=np.float32), device=dev)
        self.p, self.m = components.shape
        self.C = prepare_bank(C, mode)
        self.params = pad(down).contiguous(), pad(up).contiguous()
        self.grads = tuple(torch.zeros_like(t) for t in self.params)
        self.low = tuple(t.to(torch.bfloat16) for t in self.params) if mode == "bf16" else self.params
        self.scale = torch.ones(G, device=dev)
        each = lambda ts: [t[g] for t in ts for g in range(G)]  # noqa: E731
        self.opt = AdamW(each(self.params), each(self.grads), lr=est.learning_rate, betas=est.betas, weight_decay=est.weight_decay,
                         state_bits=est.state_bits, copies=each(self.low) if mode == "bf16" else None, seed=est._seed)
        if state is not None:
            self.opt.load_state_dict({k: torch.as_tensor(v).view(self.opt.state[k].dtype) for k, v in state.items()})

    def arrays(self):
        down, up = (t.cpu().numpy() for t in self.params)
        return np.ascontiguousarray(down[..., :self.m]), np.ascontiguousarray(up[..., :self.p])

    def state(self):
        import torch

        return {k: (v.view(torch.uint8) if v.element_size() == 1 else v).cpu().numpy() for k, v in self.opt.state_dict().items()}


class AdaptedGaussianProjection(GaussianRandomProjection):
    """``GaussianRandomProjection`` with ``n_adapters`` learned adapters of rank ``rank`` beside the shared components.

    ``transform(X, adapters)`` projects row i as ``C x_i + alpha / rank * up[a]^T (down[a] x_i)`` with ``a = adapters[i]`` (-1: the shared
    projection alone; without ``adapters`` the whole call is the base class's). ``partial_fit(X, Y, adapters)`` takes one AdamW step
    per ``chunk_rows`` rows on the mean over the chunk's rows of ``||transform(x_i) - y_i||^2``, for the adapters that have rows in it; the
    components stay as they are. ``down_`` starts Gaussian with variance 1 / n_features and ``up_`` at zero, so a new adapter changes nothing.

    compute: "fp32" (also "auto") or "bf16" for the adapted products, both summed and returned in float32. state_bits: 32 or 8, how the
    optimizer holds its moments; seed: of the random rounding to 8 bits. What ``set_params`` changes after ``fit`` holds from the next call
    on, but for the adapters' number, rank and seed, which are as fitted, and ``compute`` and
    ``state_bits``, which cannot change once a step was taken."""

    def __init__(self, n_components="auto", *, n_adapters=1, rank=8, alpha=None, learning_rate=1e-3, betas=(0.9, 0.999),
                 weight_decay=0.0, state_bits=32, seed=0, eps=0.1, compute_inverse_components=False, random_state=None, device=0,
                 compute="auto", chunk_rows=65536):
        super().__init__(n_components=n_components, eps=eps, compute_inverse_components=compute_inverse_components,
                         random_state=random_state, device=device, compute=compute, chunk_rows=chunk_rows)
        self.n_adapters = n_adapters
        self.rank = rank
        self.alpha = alpha
        self.learning_rate = learning_rate
        self.betas = betas
        self.weight_decay = weight_decay
        self.state_bits = state_bits
        self.seed = seed

    def _mode(self):
        if self.compute not in ("auto", "fp32", "bf16"):
            raise ValueError("compute must be 'auto', 'fp32' or 'bf16' for adapted products")
        return "bf16" if self.compute == "bf16" else "fp32"

    def _scale(self):
        rank = self._down.shape[1]
        return float((rank if self.alpha is None else self.alpha) / rank)

    def _made_for(self):
        return self.device, self._mode(), self.state_bits

    def fit(self, X, y=None):
        from .adapters import MAX_ADAPTERS, MAX_RANK

        if not (1 <= self.rank <= MAX_RANK and 1 <= self.n_adapters <= MAX_ADAPTERS):
            raise ValueError(f"rank must lie in 1 .. {MAX_RANK} and n_adapters in 1 .. {MAX_ADAPTERS}")
        self._mode()
        super().fit(X, y)
        p, m = self.components_.shape
        # a stream of its own: the components are those of the base class for the same random_state
        rng = check_random_state(None if self.random_state is None else np.random.RandomState(check_random_state(
            self.random_state).randint(2 ** 31 - 1)))
        self._down = rng.normal(0, m ** -0.5, (self.n_adapters, self.rank, m)).astype(np.float32)
        self._up = np.zeros((self.n_adapters, self.rank, p), np.float32)
        self._seed = int(self.seed)
        self._bank, self._state, self._state_of = None, None, None
        return self

    def _on_device(self):
        from .gaussian import _torch

        _torch()
        if self._bank is not None and self._bank.made_for != self._made_for():  # another device or compute type since
            self.__dict__.update(self._held())
        if self._bank is None:
            if self._state is not None and self._state_of != (self._mode(), self.state_bits):
                raise ValueError("compute and state_bits cannot change once a step was taken: fit again")
            self._bank = _Bank(self, self.components_, self._down, self._up, self._state)
        bank = self._bank
        bank.scale.fill_(self._scale())
        bank.opt.lr, bank.opt.betas, bank.opt.weight_decay = self.learning_rate, tuple(self.betas), self.weight_decay
        return bank

    def _held(self):
        """What the bank on the device holds, as the attributes that a new one starts from."""
        (down, up), state = self._bank.arrays(), self._bank.state()
        return {"_down": down, "_up": up, "_state": state if state["steps"].any() else None, "_state_of": self._bank.made_for[1:],
                "_bank": None}

    @property
    def down_(self):
        check_is_fitted(self)
        return self._down if self._bank is None else self._bank.arrays()[0]

    @property
    def up_(self):
        check_is_fitted(self)
        return self._up if self._bank is None else self._bank.arrays()[1]

    def _ids(self, adapters, n):
        ids = np.asarray(adapters)
        if ids.shape != (n,) or ids.dtype.kind not in "iu":
            raise ValueError(f"adapters must hold one whole number for each of the {n} rows, got {ids.dtype} {ids.shape}")
        if n and (ids.min() < -1 or ids.max() >= len(self._down)):
            raise ValueError(f"adapters must lie in -1 .. {len(self._down) - 1}")
        return ids.astype(np.int32)

    def _chunks(self, X, ids, mode):
        import scipy.sparse as sp
        import torch

        dev = torch.device("cuda", self.device)
        dt = torch.bfloat16 if mode == "bf16" else torch.float32
        for s in range(0, X.shape[0], self.chunk_rows):
            blk = X[s:s + self.chunk_rows]
            blk = blk.toarray() if sp.issparse(blk) else blk
            xb = torch.as_tensor(np.ascontiguousarray(blk, dtype=np.float32), device=dev).to(dt)
            yield s, xb, torch.as_tensor(ids[s:s + self.chunk_rows], device=dev)

    def transform(self, X, adapters=None):
        if adapters is None:
            return super().transform(X)
        from .adapters import adapted_project_device

        check_is_fitted(self)
        X = validate_data(self, X, accept_sparse=["csr"], reset=False, dtype=[np.float64, np.float32])
        ids, mode = self._ids(adapters, X.shape[0]), self._mode()
        bank = self._on_device()
        out = np.empty((X.shape[0], bank.p), np.float32)
        for s, xb, ib in self._chunks(X, ids, mode):
            y = adapted_project_device(xb, bank.C, *bank.low, ib, scale=bank.scale, compute=mode, prepared=True)
            out[s:s + xb.shape[0]] = y.cpu().numpy()
        return out

    def partial_fit(self, X, Y, adapters):
        """One step per chunk towards the targets Y (n x n_components). The first call fits the components to X's width if that was not
        done. ``loss_``: the last chunk's mean squared distance before its step."""
        from .adapters import adapted_project_backward_device, adapted_project_device

        if not hasattr(self, "components_"):
            self.fit(X)
        X = validate_data(self, X, accept_sparse=["csr"], reset=False, dtype=[np.float64, np.float32])
        ids, mode = self._ids(adapters, X.shape[0]), self._mode()
        Y = check_array(Y, dtype=np.float32)
        if Y.shape != (X.shape[0], self.components_.shape[0]):
            raise ValueError(f"Y must have shape {(X.shape[0], self.components_.shape[0])}, got {Y.shape}")
        import torch

        bank = self._on_device()
        kw = dict(scale=bank.scale, compute=mode, prepared=True)
        grads = bank.grads[0][..., :bank.m], bank.grads[1][..., :bank.p]
        for s, xb, ib in self._chunks(X, ids, mode):
            target = torch.as_tensor(Y[s:s + xb.shape[0]], device=xb.device)
            y, hidden = adapted_project_device(xb, bank.C, *bank.low, ib, return_hidden=True, **kw)
            off = y - target
            adapted_project_backward_device((off * (2.0 / xb.shape[0])).to(xb.dtype), xb, None, *bank.low, ib, hidden, out=grads, **kw)
            has = torch.zeros(len(self._down) + 1, dtype=torch.uint8, device=xb.device)
            has[ib.long()] = 1  # -1: the entry behind the last
            bank.opt.step(has[:-1].repeat(2))
            self.loss_ = float(off.square().sum(1).mean())
        return self

    def __getstate__(self):
        state = dict(super().__getstate__())
        if state.get("_bank") is not None:  # device memory does not travel: what it holds does
            state.update(self._held())
        return state

    def __setstate__(self, state):
        self.__dict__.update(state)
        if "_down" in state and "_seed" not in state:  # a pickle of an estimator that did not keep the seed of its fit
            self._seed = int(self.seed)
