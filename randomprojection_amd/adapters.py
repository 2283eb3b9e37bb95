"""Low-rank adapters of many requests beside the dense projection, and their gradients.

``gaussian.dense_project_device`` projects every row by one frozen matrix C (p x m). Here G adapters of rank R
stand beside it, in two banks with the long axis contiguous: ``down`` (G x R x m) and ``up`` (G x R x p). Row i
of X belongs to the adapter ``a = ids[i]`` (a row whose id is outside 0 .. G-1 has none):

    hidden_i = down[a] x_i            y_i = C x_i + scale[a] up[a]^T hidden_i

so one call serves rows of many tenants, each with a small learned part of its own, whether a request
brings one row or many. The backward pass gives the gradients of the banks and, where wanted, of X; C is
frozen and has none. An adapter of a smaller rank is padded with zero rows, which stay zero in training.

"bf16" takes X, C and the banks in bfloat16, "fp32" in float32; products are exact and summed in float32 in both,
and Y, hidden and the banks' gradients are float32 (no reference counterpart; csrc/rp_adapt.hip).
"""
from __future__ import annotations

import functools

import torch

from . import _native as nat
from .gaussian import _STEP, stream_of

__all__ = ["adapted_project_device", "adapted_project_backward_device", "prepare_bank", "MAX_RANK", "MAX_ADAPTERS"]

MAX_RANK, MAX_ADAPTERS = 128, 16383
_CODE = {"bf16": nat.RP_BF16, "fp32": nat.RP_F32}
_TYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _dtype(compute):
    try:
        return _TYPE[compute]
    except KeyError:
        raise ValueError("compute must be 'fp32' or 'bf16'") from None


def raw_stream(device):
    """The handle of torch's current stream on a device; through torch's own accessor where it has one, since making a Stream
    object costs as much as a kernel launch."""
    get = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return get(device) if get is not None else torch.cuda.current_stream(device).cuda_stream


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(code, n, m, p, G, R, what):
    return nat.load().rp_adapt_workspace_bytes(code, n, m, p, G, R, what)


def prepare_bank(W, compute: str):
    """W cast to the compute type, contiguous, its last axis padded with zeros to the kernels' multiple: what
    ``prepared=True`` expects of C, Ct, down and up. Returned as it is where it is all that already."""
    W = W.to(_dtype(compute))
    pad = -W.shape[-1] % _STEP[compute]
    if pad:
        W = torch.nn.functional.pad(W, (0, pad))
    W = W.contiguous()
    return W if W.data_ptr() % 16 == 0 else W.clone()


def _rows(X, compute):
    """X as the library takes it: of the compute type, with a row stride of its own, rows aligned unless their width needs
    padding (the library copies them then); else a copy."""
    if X.dtype is _TYPE[compute]:
        row, one = X.stride()
        if one == 1 and (row >= X.shape[1] or X.shape[0] <= 1) and (
                X.shape[1] % _STEP[compute] or (X.data_ptr() % 16 == 0 and row * X.element_size() % 16 == 0)):
            return X
    X = X.to(_TYPE[compute]).contiguous()
    return X if X.data_ptr() % 16 == 0 else X.clone()


def _ld(X):
    return max(X.stride(0), X.shape[1])


def _operand(name, W, shape, compute, prepared):
    """``shape``: the expected sizes, the last one before padding."""
    if prepared:
        want = (*shape[:-1], shape[-1] + -shape[-1] % _STEP[compute])
        if W.shape != want or W.dtype is not _TYPE[compute] or not W.is_contiguous() or W.data_ptr() % 16:
            raise ValueError(f"prepared {name} must be a contiguous 16-byte aligned {_dtype(compute)} tensor of shape "
                             f"{want}, got {W.dtype} {tuple(W.shape)}")
        return W
    if W.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(W.shape)}")
    return prepare_bank(W, compute)


def _check_common(X, down, up, ids, scale, compute):
    _dtype(compute)
    if X.dim() != 2 or down.dim() != 3 or up.dim() != 3:
        raise ValueError("X must be 2-D, down and up 3-D (adapters, rank, width)")
    (n, m), (G, R, _), (G2, R2, _) = X.shape, down.shape, up.shape
    if G != G2 or R != R2 or not G or not R or not m:
        raise ValueError(f"down {tuple(down.shape)} and up {tuple(up.shape)} must have the same, positive, number of "
                         "adapters and rank")
    if R > MAX_RANK or G > MAX_ADAPTERS:
        raise ValueError(f"at most {MAX_ADAPTERS} adapters of rank {MAX_RANK}, got {G} of rank {R}")
    if ids.dtype is not torch.int32 or ids.shape != (n,) or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int32 tensor of {n} entries, got {ids.dtype} {tuple(ids.shape)}")
    if scale is not None and (scale.dtype is not torch.float32 or scale.shape != (G,) or not scale.is_contiguous()):
        raise ValueError("scale must be a contiguous float32 tensor with one entry for each adapter")
    return n, m, G, R


def _check_device(*tensors):
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")
    if dev.type != "cuda":
        raise RuntimeError("adapted projections need an MI355X (no CPU fallback)")
    return dev


def _on_stream(stream, dev, tensors):
    """The stream to launch on. One other than torch's current stream waits for what is queued there (casts of the
    operands), and the temporaries made here are kept for it."""
    now = raw_stream(dev.index)
    if stream is None or stream == now:
        return now
    cur = torch.cuda.current_stream(dev)
    ext = stream_of(stream, dev)
    ext.wait_stream(cur)
    for t in tensors:
        if t is not None:
            t.record_stream(ext)
    return stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _strided(name, t, shape, dtype):
    if t.dtype is not dtype or t.shape != shape or t.stride(-1) != 1 or any(
            t.stride(d) < t.stride(d + 1) * t.shape[d + 1] for d in range(t.dim() - 1)):
        raise ValueError(f"{name} must be a {dtype} tensor of shape {shape} with unit column stride and rows that do not overlap")
    return t


def _share(a, b):
    """Whether two tensors, unit column strides or contiguous, hold a byte in common. Rows side by side in one buffer (same row stride,
    columns apart) do not, though they lie between each other."""
    if not a.numel() or not b.numel():
        return False
    span = lambda t: sum((k - 1) * s for k, s in zip(t.shape, t.stride())) * t.element_size() + t.element_size()  # noqa: E731
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + span(a) <= pb or pb + span(b) <= pa:
        return False
    row = a.stride(-2) * a.element_size() if a.dim() > 1 else 0
    for t in (a, b):
        if not row or t.dim() < 2 or t.stride(-1) != 1 or any(s * t.element_size() % row for s, k in zip(t.stride()[:-1], t.shape) if k > 1):
            return True
    at, wide = (pb - pa) % row, [t.shape[-1] * t.element_size() for t in (a, b)]
    return at < wide[0] or at + wide[1] > row


def _own_memory(name, out, *read):
    for t in read:
        if t is not None and _share(out, t):
            raise ValueError(f"{name} must not share memory with what the call reads or its other output")


def adapted_project_device(X, C, down, up, ids, *, scale=None, out=None, compute: str = "fp32", stream=None,
                           prepared: bool = False, return_hidden: bool = False):
    """``X @ C.T`` plus each row's adapter for device tensors X (n x m), C (p x m), down (G x R x m), up (G x R x p) and
    int32 ids (n); scale: float32 (G), 1 if None. Returns Y (n x p, float32), or (Y, hidden) with the n x R hidden
    that the backward pass takes. ``prepared``: C, down and up already went through ``prepare_bank`` for this compute
    mode. ``out``: a float32 n x p tensor with unit column stride to write to. Runs on ``stream`` (a raw handle;
    default: torch's current stream), without synchronising; it can be captured into a graph."""
    n, m, G, R = _check_common(X, down, up, ids, scale, compute)
    if C.dim() != 2:
        raise ValueError("C must be 2-D")
    p = C.shape[0]
    Cc = _operand("C", C, (p, m), compute, prepared)
    Dc = _operand("down", down, (G, R, m), compute, prepared)
    Uc = _operand("up", up, (G, R, p), compute, prepared)
    if out is not None:
        _own_memory("out", _strided("out", out, (n, p), torch.float32), X, C, down, up, ids, scale)
    dev = _check_device(X, C, down, up, ids, scale, out)
    Xc = _rows(X, compute)
    y = out if out is not None else torch.empty(n, p, dtype=torch.float32, device=dev)
    hidden = torch.empty(n, R, dtype=torch.float32, device=dev) if return_hidden else None
    if n:
        lib, code = nat.load(), _CODE[compute]
        need = _workspace_bytes(code, n, m, p, G, R, nat.RP_ADAPT_PROJECT)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        st = _on_stream(stream, dev, (Xc, Cc, Dc, Uc, ids, scale, y, hidden, ws))
        nat.check(lib.rp_adapt_project_device(
            dev.index, Xc.data_ptr(), _ld(Xc), code, n, m, Cc.data_ptr(), p, Dc.data_ptr(), Uc.data_ptr(), G, R, _ptr(scale),
            ids.data_ptr(), y.data_ptr(), max(y.stride(0), p), _ptr(hidden), ws.data_ptr(), need, st))
    return (y, hidden) if return_hidden else y


def adapted_project_backward_device(dY, X, Ct, down, up, ids, hidden, *, scale=None, out=None, compute: str = "fp32",
                                    stream=None, prepared: bool = False):
    """The gradients of ``adapted_project_device``: (dX, d_down, d_up) for dY (n x p), the forward pass's X, ids and
    hidden, and Ct = C.T (m x p). dX has the compute type; with Ct None it is left out (None is returned in its place).
    d_down (G x R x m) and d_up (G x R x p) are float32, zeros for adapters without rows; ``out``: a pair of such
    tensors (unit column stride) to write them to. ``prepared``: Ct, down and up went through ``prepare_bank``.
    The same call gives the same bits. Runs on ``stream`` as the forward pass does."""
    n, m, G, R = _check_common(X, down, up, ids, scale, compute)
    if dY.dim() != 2 or dY.shape[0] != n or 0 in dY.shape[1:]:
        raise ValueError(f"dY must be 2-D with {n} rows, got {tuple(dY.shape)}")
    p = dY.shape[1]
    if hidden.dtype is not torch.float32 or hidden.shape != (n, R) or not hidden.is_contiguous():
        raise ValueError(f"hidden must be the contiguous float32 ({n}, {R}) tensor of the forward pass")
    Tc = None if Ct is None else _operand("Ct", Ct, (m, p), compute, prepared)
    Dc = _operand("down", down, (G, R, m), compute, prepared)
    Uc = _operand("up", up, (G, R, p), compute, prepared)
    if out is not None:
        d_down, d_up = _strided("out[0]", out[0], (G, R, m), torch.float32), _strided("out[1]", out[1], (G, R, p), torch.float32)
        for i, t in enumerate((d_down, d_up)):
            _own_memory(f"out[{i}]", t, X, dY, Ct, down, up, ids, hidden, scale, d_up if i == 0 else None)
    dev = _check_device(X, dY, Ct, down, up, ids, hidden, scale, *(out or ()))
    Xc, Yc = _rows(X, compute), _rows(dY, compute)
    if out is None:
        d_down, d_up = (torch.empty(G, R, w, dtype=torch.float32, device=dev) for w in (m, p))
        strides = m, R * m, p, R * p
    else:
        row = lambda t: max(t.stride(1), t.shape[2])  # noqa: E731
        strides = tuple(x for t in (d_down, d_up) for x in (row(t), max(t.stride(0), row(t) * R)))
    dX = None if Ct is None else torch.empty(n, m, dtype=_dtype(compute), device=dev)
    lib, code = nat.load(), _CODE[compute]
    what = nat.RP_ADAPT_GRADIENTS if dX is None else nat.RP_ADAPT_GRADIENTS_DX
    need = _workspace_bytes(code, n, m, p, G, R, what)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    st = _on_stream(stream, dev, (Xc, Yc, Tc, Dc, Uc, ids, hidden, scale, dX, d_down, d_up, ws))
    nat.check(lib.rp_adapt_gradients_device(
        dev.index, Yc.data_ptr(), _ld(Yc), Xc.data_ptr(), _ld(Xc), code, n, m, p, _ptr(Tc) if n else None, Dc.data_ptr(),
        Uc.data_ptr(), G, R, _ptr(scale), ids.data_ptr(), hidden.data_ptr(), _ptr(dX) if n else None, m, d_down.data_ptr(),
        *strides[:2], d_up.data_ptr(), *strides[2:], ws.data_ptr(), need, st))
    return dX, d_down, d_up
