"""Adam with the interface and state layout of ``torch.optim.Adam`` (the optimizer the reference
builds at train.py:131-136), stepping every parameter in ONE multi-tensor HIP kernel launch.

The per-parameter step counts live on the device (like torch's ``capturable=True`` mode) and the
descriptor table travels in the kernel arguments, so ``step()`` makes no host<->device copy and no
synchronisation: it can be captured into a HIP graph and replayed."""
from __future__ import annotations

import array
import ctypes
import math

import torch

from . import _lib
from ._lib import call


class _Desc(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("g", ctypes.c_void_p), ("m", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("step", ctypes.c_void_p), ("n", ctypes.c_int64)]


DESC_BYTES = ctypes.sizeof(_Desc)


def build_table(rows):
    """rows: list of (p_ptr, g_ptr, m_ptr, v_ptr, step_ptr, n).  Returns a host ctypes array (of ``_Desc``, whose fields are
    all 64 bits wide: one flat array, a third of the time of a structure per row)."""
    flat = array.array("Q", [x or 0 for row in rows for x in row])
    return (ctypes.c_char * (8 * len(flat))).from_buffer(flat)


def _grad_rows(grads, what):
    """(rows of ``build_table``, the tensors they point to, their device): every storage once, empty tensors left out,
    copies of tensors that are not dense."""
    rows, keep, seen, device = [], [], set(), None
    for g in grads:
        if g.is_sparse or not g.is_cuda or g.dtype != torch.float32:
            raise RuntimeError(f"{what}: gradients must be dense float32 device tensors, got {g.dtype} on {g.device}")
        if device is not None and g.device != device:
            raise RuntimeError(f"{what}: gradients on {device} and {g.device}")
        device = g.device
        if g.numel() == 0 or (g.data_ptr(), g.numel()) in seen:
            continue
        seen.add((g.data_ptr(), g.numel()))
        dense = g if g.is_contiguous() else g.contiguous()
        keep.append((g, dense))
        rows.append((None, dense.data_ptr(), None, None, None, g.numel()))
    return rows, keep, device


def _norm_into(rows, out, scale, max_norm):
    """out[0] = the norm, out[1] = the multiplier; returns the table and the workspace (the clipped Adam step uses them
    again)."""
    table = build_table(rows)
    nbytes = _lib.load().eeggan_grad_norm_workspace(table, len(rows))
    ws = torch.empty(max(nbytes, 16), device=out.device, dtype=torch.uint8)
    call("eeggan_grad_norm", table, len(rows), float(scale), float(max_norm), out.data_ptr(), ws.data_ptr(), nbytes,
         torch.cuda.current_stream().cuda_stream)
    return table, ws


def _grads_of(parameters):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [p.grad for p in parameters if p.grad is not None]


def grad_norm(grads):
    """sqrt of the sum of squares of all elements of ``grads`` (tensors; float32), as a 0-dim device tensor: one pass
    over them, in double, no synchronisation.  A tensor that is listed twice counts once."""
    rows, _keep, device = _grad_rows([grads] if isinstance(grads, torch.Tensor) else list(grads), "grad_norm")
    if not rows:
        return torch.zeros((), device=device if device is not None else "cuda")
    out = torch.empty(2, device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        _norm_into(rows, out, 1.0, math.inf)
    return out[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """``torch.nn.utils.clip_grad_norm_`` on this package's kernels (``foreach`` has no effect): scales the gradients of
    ``parameters`` in place so that their global 2-norm is at most ``max_norm`` (multiplier
    min(1, max_norm / (norm + 1e-6))) and returns the norm they had, a 0-dim device tensor.  Nothing waits for the device unless ``error_if_nonfinite`` asks for the check; a
    norm below the bound costs no second pass over the gradients.  ``Adam(max_grad_norm=...)`` needs no call of this:
    its step reads the multiplier and never writes clipped gradients."""
    if float(norm_type) != 2.0:
        raise NotImplementedError("clip_grad_norm_: only the 2-norm is supported")
    if not float(max_norm) > 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm {max_norm} is not positive")
    rows, keep, device = _grad_rows(_grads_of(parameters), "clip_grad_norm_")
    if not rows:
        return torch.zeros((), device=device if device is not None else "cuda")
    out = torch.empty(2, device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        table, _ws = _norm_into(rows, out, 1.0, max_norm)
        if error_if_nonfinite and not math.isfinite(float(out[0])):
            raise RuntimeError(f"clip_grad_norm_: the total norm is {float(out[0])}; gradients are left as they are")
        call("eeggan_grad_scale", table, len(rows), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
        for g, dense in keep:
            if dense is not g:
                g.copy_(dense)
    return out[0]


class Adam(torch.optim.Optimizer):
    """``max_grad_norm``: bound of the global 2-norm of the gradients of a step (all parameter groups together, after
    ``grad_scale``); the step then uses min(1, max_grad_norm / (norm + 1e-6)) times the gradients, which stay as they
    are in ``p.grad``, and ``grad_norm`` holds the norm it found (a 0-dim device tensor that every step, captured ones
    included, rewrites).  The bound is an attribute like ``grad_scale``: copies and pickles of the optimizer have it, its
    ``state_dict`` (torch's layout) does not."""

    max_grad_norm = _norm = None  # (for objects that were pickled without them)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False, max_grad_norm=None):
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError(f"Adam: max_grad_norm {max_grad_norm} is not positive")
        if weight_decay != 0 or amsgrad:
            raise NotImplementedError("Adam: weight_decay and amsgrad are not supported")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=0, amsgrad=False))
        self.grad_scale = 1.0  # set to 1/world_size when gradients arrive as a sum over ranks
        self.max_grad_norm = max_grad_norm
        self._norm = None  # device: (norm, multiplier) of the last clipped step

    def __getstate__(self):
        """Copies and pickles keep the bound and the gradients' scale (the base class keeps groups and state only); the norm
        of the last step is not taken along."""
        own = {k: self.__dict__[k] for k in ("grad_scale", "max_grad_norm") if k in self.__dict__}
        return dict(super().__getstate__(), **own)

    @property
    def grad_norm(self):
        """Norm of the gradients of the last step with ``max_grad_norm`` (None before the first one)."""
        return None if self._norm is None else self._norm[0]

    def _init_state(self, p):
        st = self.state[p]
        if len(st) == 0:
            st["step"] = torch.zeros((), device=p.device, dtype=torch.float32)
            st["exp_avg"] = torch.zeros_like(p)
            st["exp_avg_sq"] = torch.zeros_like(p)
        elif not st["step"].is_cuda:  # state restored from a checkpoint written by torch.optim.Adam
            st["step"] = st["step"].to(device=p.device, dtype=torch.float32)
        return st

    @torch.no_grad()
    def step(self, closure=None, grads=None):
        """``grads`` optionally maps a parameter to the tensor holding its gradient (e.g. a slice of
        an all-reduced bucket); by default ``p.grad`` is used and parameters without one are skipped."""
        if closure is not None:
            raise NotImplementedError("Adam.step: closures are not supported")
        from . import ops
        work = []  # (group, rows) with the gradient tensors kept alive until everything is launched
        keep = []
        for group in self.param_groups:
            rows = []
            for p in group["params"]:
                g = grads.get(p) if grads is not None else p.grad
                if g is None:
                    continue
                if grads is not None and (g.numel() != p.numel() or g.dtype != p.dtype or g.device != p.device):
                    raise RuntimeError(f"Adam: a gradient of {g.numel()} elements, {g.dtype} on {g.device}, for a parameter of "
                                       f"{p.numel()}, {p.dtype} on {p.device}")
                if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous():
                    raise RuntimeError("Adam: parameters must be contiguous float32 device tensors")
                if not g.is_contiguous():
                    g = g.contiguous()
                st = self._init_state(p)
                rows.append((p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(),
                             st["step"].data_ptr(), p.numel()))
                keep.append(g)
            if rows:
                work.append((group, rows))
        if not work:
            return None
        if self.max_grad_norm is not None:
            self._clipped_step(work, keep)
        else:
            for group, rows in work:
                b1, b2 = group["betas"]
                call("eeggan_adam_step", build_table(rows), len(rows), float(group["lr"]), float(b1), float(b2),
                     float(group["eps"]), float(self.grad_scale), torch.cuda.current_stream().cuda_stream)
        ops.bump_weights_epoch()  # cached derived weight views are stale from here on
        return None

    def _clipped_step(self, work, grads):
        work = [(group, rows) for group, rows in ((group, [r for r in rows if r[5]]) for group, rows in work) if rows]
        if not work:  # (tensors without elements)
            return
        device = grads[0].device
        if len({(g.dtype, g.get_device()) for g in grads} | {(torch.float32, device.index)}) != 1:
            found = sorted({f"{g.dtype} on {g.device}" for g in grads})
            raise RuntimeError(f"Adam: gradients of {', '.join(found)}, expected float32 on one device")
        if self._norm is None or self._norm.device != device:
            self._norm = torch.zeros(2, device=device, dtype=torch.float32)
        with torch.cuda.device(device):
            # (one norm over the gradients of all groups, whose tensors lie one group after the other in the table)
            table, ws = _norm_into([row for _, rows in work for row in rows], self._norm, self.grad_scale,
                                   self.max_grad_norm)
            first, stream = ctypes.addressof(table), torch.cuda.current_stream().cuda_stream
            for group, rows in work:
                b1, b2 = group["betas"]
                call("eeggan_adam_step_clipped", first, len(rows), float(group["lr"]), float(b1), float(b2),
                     float(group["eps"]), self._norm.data_ptr(), ws.data_ptr(), ws.numel(), stream)
                first += len(rows) * DESC_BYTES
