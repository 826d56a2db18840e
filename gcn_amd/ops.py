"""Tensor-level operators over libccnn_hip.so.

Each function takes CUDA (ROCm) torch tensors, checks shapes/dtypes on the host
so that a kernel never sees an operand it was not written for, and enqueues the
work on torch's current stream.  Names follow the reference's kernel groups:
gather (preprocessing), forward (the test loop), sgd, mbgd_grad, update.
"""
import ctypes as C
import os
from typing import NamedTuple, Optional

import torch

from . import lib as _l

_F32, _F64 = torch.float32, torch.float64


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _req(t, dtype, name, numel=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    return t


def _sfx(dtype):
    if dtype == _F32:
        return "f32", 4
    if dtype == _F64:
        return "f64", 8
    raise TypeError(f"unsupported dtype {dtype}")


_WS_BYTES = {}


def _mbgd_ws_bytes(lib, B, z, es):
    """ccnn_mbgd_workspace_bytes, remembered (the training loop asks on every step).  The size depends
    on which implementation of the step the library picks, and CCNN_MBGD_PATH / CCNN_TILE_WAVES can
    override that."""
    k = (B, z, es, os.environ.get("CCNN_MBGD_PATH"), os.environ.get("CCNN_TILE_WAVES"))
    n = _WS_BYTES.get(k)
    if n is None:
        n = _WS_BYTES[k] = lib.ccnn_mbgd_workspace_bytes(B, z, es)
    return n


class Workspace:
    """A reusable device scratch buffer (grown on demand, never shrunk)."""

    def __init__(self, device="cuda"):
        self.device = device
        self.buf = None

    def get(self, nbytes):
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=self.device)
        return self.buf


def gather(scene, idx9, x, y, z, out=None, workspace=None, sort=True):
    """scene: flat [z*y*x] (x fastest); idx9 int32 [n, 9] -> cubes [n, 9z].
    sort=True lets the library visit the samples in centre-pixel order (same result, fewer reads)."""
    sfx, _ = _sfx(scene.dtype)
    _req(scene, scene.dtype, "scene", x * y * z)
    _req(idx9, torch.int32, "idx9")
    n = idx9.numel() // 9
    if idx9.numel() != n * 9:
        raise ValueError("idx9 must hold 9 indices per sample")
    if out is None:
        out = torch.empty((n, 9 * z), dtype=scene.dtype, device=scene.device)
    _req(out, scene.dtype, "out", n * 9 * z)
    lib = _l.load()
    ws, ws_bytes = None, 0
    if sort:
        ws_bytes = lib.ccnn_gather_workspace_bytes(n)
        if ws_bytes:
            ws = (workspace or Workspace(scene.device)).get(ws_bytes)
    fn = getattr(lib, f"ccnn_gather_{sfx}")
    _l.check(fn(_ptr(scene), _ptr(idx9), n, x, y, z, _ptr(out), _ptr(ws), ws.numel() if ws is not None else 0,
                _stream()), f"ccnn_gather_{sfx}")
    return out


class GatherPlan:
    """One sample list prepared for repeated gathers (other scenes, other passes):
    `GatherPlan(idx9, x, y)` looks at the list once; `plan.gather(scene, z)` then runs only the
    gather kernel - tiles staged in LDS (`plan.dense`) for densely labelled lists of plain 3x3
    neighbourhoods, the ordered-list kernel otherwise.  Holds its own workspace; idx9 must stay
    alive and unchanged."""

    def __init__(self, idx9, x, y):
        _req(idx9, torch.int32, "idx9")
        self.idx9, self.x, self.y = idx9, x, y
        self.n = idx9.numel() // 9
        if idx9.numel() != self.n * 9:
            raise ValueError("idx9 must hold 9 indices per sample")
        lib = _l.load()
        nbytes = lib.ccnn_gather_plan_workspace_bytes(self.n, x, y)
        self.ws = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=idx9.device)
        self._h = C.c_void_p()
        _l.check(lib.ccnn_gather_plan_create(_ptr(idx9), self.n, x, y, _ptr(self.ws), self.ws.numel(), _stream(),
                                             C.byref(self._h)), "ccnn_gather_plan_create")
        self.dense = lib.ccnn_gather_plan_kind(self._h) == 1

    def gather(self, scene, z, out=None):
        sfx, _ = _sfx(scene.dtype)
        _req(scene, scene.dtype, "scene", self.x * self.y * z)
        if out is None:
            out = torch.empty((self.n, 9 * z), dtype=scene.dtype, device=scene.device)
        _req(out, scene.dtype, "out", self.n * 9 * z)
        fn = getattr(_l.load(), f"ccnn_gather_planned_{sfx}")
        _l.check(fn(self._h, _ptr(scene), z, _ptr(out), _stream()), f"ccnn_gather_planned_{sfx}")
        return out

    def __del__(self):
        if getattr(self, "_h", None) and _l is not None:      # module globals are gone at interpreter exit
            _l.load().ccnn_gather_plan_destroy(self._h)
            self._h = None


def forward(params, cubes, z, want_probs=True, want_argmax=True, workspace=None):
    """Test-loop forward over cubes [n, 9z] -> (probs [n, classes] | None, argmax int32 [n] | None).
    z: the band count, or lib.geometry(z, n_classes) for a class count other than 13 (here and below)."""
    sfx, es = _sfx(params.dtype)
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    n = cubes.numel() // d.cube
    _req(cubes, params.dtype, "cubes", n * d.cube)
    probs = torch.empty((n, d.n_classes), dtype=params.dtype, device=params.device) if want_probs else None
    argmax = torch.empty(n, dtype=torch.int32, device=params.device) if want_argmax else None
    if n == 0:
        return probs, argmax
    lib = _l.load()
    nbytes = lib.ccnn_forward_workspace_bytes(n, z, es)
    ws = (workspace or Workspace(params.device)).get(nbytes)
    fn = getattr(lib, f"ccnn_forward_{sfx}")
    _l.check(fn(_ptr(params), _ptr(cubes), n, z, _ptr(probs), _ptr(argmax), _ptr(ws), ws.numel(), _stream()),
             f"ccnn_forward_{sfx}")
    return probs, argmax


def forward_logits(params, cubes, z, workspace=None):
    """The test-loop forward up to its last layer: logits [n, classes], for log_probs."""
    sfx, es = _sfx(params.dtype)
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    n = cubes.numel() // d.cube
    _req(cubes, params.dtype, "cubes", n * d.cube)
    logits = torch.empty((n, d.n_classes), dtype=params.dtype, device=params.device)
    if n == 0:
        return logits
    lib = _l.load()
    ws = (workspace or Workspace(params.device)).get(lib.ccnn_forward_workspace_bytes(n, z, es))
    fn = getattr(lib, f"ccnn_forward_logits_{sfx}")
    _l.check(fn(_ptr(params), _ptr(cubes), n, z, _ptr(logits), None, _ptr(ws), ws.numel(), _stream()),
             f"ccnn_forward_logits_{sfx}")
    return logits


def forward_scene(params, scene, idx9, x, y, z, want_probs=True, want_argmax=True, workspace=None):
    """forward() on pixels of the scene: idx9 int32 [n, 9] neighbour lists; no cubes are stored."""
    sfx, es = _sfx(params.dtype)
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    _req(scene, params.dtype, "scene", x * y * d.z)
    _req(idx9, torch.int32, "idx9")
    n = idx9.numel() // 9
    if idx9.numel() != n * 9:
        raise ValueError("idx9 must hold 9 indices per sample")
    probs = torch.empty((n, d.n_classes), dtype=params.dtype, device=params.device) if want_probs else None
    argmax = torch.empty(n, dtype=torch.int32, device=params.device) if want_argmax else None
    if n == 0:
        return probs, argmax
    lib = _l.load()
    ws = (workspace or Workspace(params.device)).get(lib.ccnn_forward_workspace_bytes(n, z, es))
    fn = getattr(lib, f"ccnn_forward_scene_{sfx}")
    _l.check(fn(_ptr(params), _ptr(scene), _ptr(idx9), n, x, y, z, _ptr(probs), _ptr(argmax), _ptr(ws), ws.numel(),
                _stream()), f"ccnn_forward_scene_{sfx}")
    return probs, argmax


def count_correct(argmax, labels):
    """Device count of argmax+1 == labels; returns a 1-element int32 tensor."""
    _req(argmax, torch.int32, "argmax")
    _req(labels, torch.int32, "labels", argmax.numel())
    count = torch.empty(1, dtype=torch.int32, device=argmax.device)
    _l.check(_l.load().ccnn_count_correct(_ptr(argmax), _ptr(labels), argmax.numel(), _ptr(count), _stream()),
             "ccnn_count_correct")
    return count


def sgd(params, cubes, onehot, first, count, z, lr, loss, workspace=None):
    """fp64 per-sample SGD over samples [first, first+count); params and the
    1-element fp64 tensor `loss` are updated in place."""
    d = _l.dims(z)
    _req(params, _F64, "params", d.nparams)
    n = cubes.numel() // d.cube
    _req(cubes, _F64, "cubes", n * d.cube)
    _req(onehot, torch.int32, "onehot", n * d.n_classes)
    _req(loss, _F64, "loss", 1)
    if first < 0 or count < 0 or first + count > n:
        raise ValueError(f"samples [{first}, {first + count}) outside [0, {n})")
    lib = _l.load()
    ws = (workspace or Workspace(params.device)).get(lib.ccnn_sgd_workspace_bytes(z))
    _l.check(lib.ccnn_sgd_f64(_ptr(params), _ptr(cubes), _ptr(onehot), first, count, z, float(lr), _ptr(loss),
                              _ptr(ws), ws.numel(), _stream()), "ccnn_sgd_f64")


def mbgd_grad(params, cubes, onehot, first, B, z, grad=None, loss_values=None, probs=None, workspace=None):
    """Batch-summed gradient of samples [first, first+B) -> (grad, loss_values[B] fp64)."""
    sfx, es = _sfx(params.dtype)
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    n = cubes.numel() // d.cube
    _req(cubes, params.dtype, "cubes", n * d.cube)
    _req(onehot, torch.int32, "onehot", n * d.n_classes)
    if B <= 0 or first < 0 or first + B > n:
        raise ValueError(f"batch [{first}, {first + B}) outside [0, {n})")
    if grad is None:
        grad = torch.empty(d.nparams, dtype=params.dtype, device=params.device)
    _req(grad, params.dtype, "grad", d.nparams)
    if loss_values is None:
        loss_values = torch.empty(B, dtype=_F64, device=params.device)
    _req(loss_values, _F64, "loss_values")
    if loss_values.numel() < B:
        raise ValueError("loss_values shorter than the batch")
    if probs is not None:
        _req(probs, params.dtype, "probs", B * d.n_classes)
    lib = _l.load()
    ws = (workspace or Workspace(params.device)).get(_mbgd_ws_bytes(lib, B, z, es))
    fn = getattr(lib, f"ccnn_mbgd_grad_{sfx}")
    _l.check(fn(_ptr(params), _ptr(cubes), _ptr(onehot), first, B, z, _ptr(grad), _ptr(loss_values), _ptr(probs),
                _ptr(ws), ws.numel(), _stream()), f"ccnn_mbgd_grad_{sfx}")
    return grad, loss_values


def mbgd_step(params, cubes, onehot, first, B, z, lr, loss_values=None, workspace=None, comm=None, divisor=None):
    """Gradient and the variant's own update in one call; params updated in place.
    comm (a gcn_amd.comm.NodeComm): the data-parallel step - this rank's B samples, the sums
    exchanged with the other ranks inside the reduction kernel; fp64 then divides by `divisor`
    (the global batch)."""
    sfx, es = _sfx(params.dtype)
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    n = cubes.numel() // d.cube
    _req(cubes, params.dtype, "cubes", n * d.cube)
    _req(onehot, torch.int32, "onehot", n * d.n_classes)
    if B <= 0 or first < 0 or first + B > n:
        raise ValueError(f"batch [{first}, {first + B}) outside [0, {n})")
    if loss_values is None:
        loss_values = torch.empty(B, dtype=_F64, device=params.device)
    _req(loss_values, _F64, "loss_values")
    if loss_values.numel() < B:
        raise ValueError("loss_values shorter than the batch")
    lib = _l.load()
    ws = (workspace or Workspace(params.device)).get(_mbgd_ws_bytes(lib, B, z, es))
    if comm is not None:
        fn = getattr(lib, f"ccnn_mbgd_step_dp_{sfx}")
        extra = () if params.dtype == torch.float32 else (int(divisor if divisor else B * comm.world),)
        _l.check(fn(comm._h, _ptr(params), _ptr(cubes), _ptr(onehot), first, B, z, float(lr), *extra,
                    _ptr(loss_values), _ptr(ws), ws.numel(), _stream()), f"ccnn_mbgd_step_dp_{sfx}")
        return loss_values
    fn = getattr(lib, f"ccnn_mbgd_step_{sfx}")
    _l.check(fn(_ptr(params), _ptr(cubes), _ptr(onehot), first, B, z, float(lr), _ptr(loss_values), _ptr(ws),
                ws.numel(), _stream()), f"ccnn_mbgd_step_{sfx}")
    return loss_values


class MbgdStepper:
    """mbgd_step for a training loop: everything that does not change from step to step (argument
    checks, workspace, pointers, the stream, the C function) is resolved once, so a step costs one
    foreign call - the host side of ops.mbgd_step is about 9 us per step, which is half of what the
    GPU needs for a step of 128 samples.  The tensors must stay alive and in place while the stepper
    is used; steps run on the stream that was current when the stepper was made.
        st = MbgdStepper(params, cubes, onehot, B, z, loss_values=ring)   # ring: [nb, B] float64 or None
        st.step(first, lr, row)                                           # loss of the step -> ring[row]
    comm / divisor as in mbgd_step (the data-parallel step)."""

    def __init__(self, params, cubes, onehot, B, z, loss_values=None, workspace=None, comm=None, divisor=None):
        sfx, es = _sfx(params.dtype)
        d = _l.dims(z)
        _req(params, params.dtype, "params", d.nparams)
        self.n = cubes.numel() // d.cube
        _req(cubes, params.dtype, "cubes", self.n * d.cube)
        _req(onehot, torch.int32, "onehot", self.n * d.n_classes)
        if B <= 0 or B > self.n:
            raise ValueError(f"batch of {B} does not fit {self.n} samples")
        if loss_values is None:
            loss_values = torch.empty((1, B), dtype=_F64, device=params.device)
        _req(loss_values, _F64, "loss_values")
        if loss_values.numel() < B or loss_values.numel() % B:
            raise ValueError("loss_values must hold whole rows of B values")
        lib = _l.load()
        self.B, self.z, self.rows = int(B), int(z), loss_values.numel() // B
        self._keep = (params, cubes, onehot, loss_values, workspace, comm)
        self._ws = (workspace or Workspace(params.device)).get(_mbgd_ws_bytes(lib, B, z, es))
        self._p, self._c, self._o = _ptr(params), _ptr(cubes), _ptr(onehot)
        self._lv, self._lv_stride = loss_values.data_ptr(), 8 * B
        self._wsp, self._wsn, self._st = _ptr(self._ws), self._ws.numel(), _stream()
        self._f32 = params.dtype == torch.float32
        if comm is not None:
            self._fn = getattr(lib, f"ccnn_mbgd_step_dp_{sfx}")
            self._comm = comm._h
            self._div = int(divisor if divisor else B * comm.world)
        else:
            self._fn = getattr(lib, f"ccnn_mbgd_step_{sfx}")
            self._comm = None
        self._what = self._fn.__name__

    def step(self, first, lr, row=0):
        if first < 0 or first + self.B > self.n or row < 0 or row >= self.rows:
            raise ValueError(f"batch [{first}, {first + self.B}) / loss row {row} out of range")
        lv = C.c_void_p(self._lv + row * self._lv_stride)
        if self._comm is None:
            rc = self._fn(self._p, self._c, self._o, first, self.B, self.z, lr, lv, self._wsp, self._wsn, self._st)
        elif self._f32:
            rc = self._fn(self._comm, self._p, self._c, self._o, first, self.B, self.z, lr, lv, self._wsp, self._wsn, self._st)
        else:
            rc = self._fn(self._comm, self._p, self._c, self._o, first, self.B, self.z, lr, self._div, lv, self._wsp,
                          self._wsn, self._st)
        if rc:
            _l.check(rc, self._what)


def update(params, grad, lr, z, divisor=None, freeze_conv_bias=True):
    """fp64: params -= lr*grad/divisor.  fp32: params -= lr*grad with the conv bias
    left untouched (the fp32 reference never updates it)."""
    d = _l.dims(z)
    _req(params, params.dtype, "params", d.nparams)
    _req(grad, params.dtype, "grad", d.nparams)
    lib = _l.load()
    if params.dtype == _F64:
        if not divisor or divisor <= 0:
            raise ValueError("fp64 update needs the batch size as divisor")
        _l.check(lib.ccnn_update_f64(_ptr(params), _ptr(grad), float(lr), int(divisor), d.nparams, _stream()),
                 "ccnn_update_f64")
    else:
        _sfx(params.dtype)
        _l.check(lib.ccnn_update_f32(_ptr(params), _ptr(grad), float(lr), z, int(bool(freeze_conv_bias)),
                                     _stream()), "ccnn_update_f32")


def update_adagrad(params, rms, grad, lr, it):
    _req(params, _F64, "params")
    _req(rms, _F64, "rms", params.numel())
    _req(grad, _F64, "grad", params.numel())
    _l.check(_l.load().ccnn_update_adagrad_f64(_ptr(params), _ptr(rms), _ptr(grad), float(lr), int(it),
                                               params.numel(), _stream()), "ccnn_update_adagrad_f64")


# ---- scoring, loss and optimiser on any model's logits, gradients and parameters ----

_TYPES = {_F32: _l.TYPE_F32, _F64: _l.TYPE_F64, torch.bfloat16: _l.TYPE_BF16, torch.float16: _l.TYPE_F16}


def _on_device(t, name, dtypes):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes:
        return t
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    raise TypeError(f"{name} has dtype {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")


def _same_device(t, name, device):
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


_T = torch.Tensor


def _refuse_list(tensors, name, dtypes):
    """Says what is wrong with a list that has to be contiguous tensors on one device."""
    for i, t in enumerate(tensors):
        _on_device(t, f"{name} {i}", dtypes)
        _same_device(t, f"{name} {i}", tensors[0].device)
        if not t.is_contiguous():
            raise ValueError(f"{name} {i} must be contiguous")


_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _called(name, like, *args):
    """What the module beside the library gives for `name`, with like's device current and that device's current
    stream.  None: an argument is not what it has to be."""
    index = like.get_device() if isinstance(like, _T) else -1
    if index < 0:
        return None
    call = getattr(_l.calls(), name)
    if index == _current():
        got = call(_raw_stream(index), index, *args)
    else:
        with torch.cuda.device(index):
            got = call(_raw_stream(index), index, *args)
    if type(got) is int:
        _l.check(got, f"ccnn_{name}")
    return got


class LogProbs(NamedTuple):
    """What log_probs returns; fp64 for fp64 logits, else fp32.  logp and entropy are rows of stats."""
    logp: torch.Tensor                   # [rows] log probability of the target
    entropy: Optional[torch.Tensor]      # [rows] in nats
    top_logp: Optional[torch.Tensor]     # [rows, top] in falling order
    top_index: Optional[torch.Tensor]    # [rows, top] int32
    stats: torch.Tensor                  # [4, rows] logp, entropy, largest logit, log sum exp(x - largest)


def _rows(t, name):
    """(rows, columns) of a matrix whose rows are contiguous and do not overlap."""
    if t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{name} must be [rows, classes] with at least one class, got {list(t.shape)}")
    rows, classes = t.shape
    if classes > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be contiguous along its classes")
    if rows > 1 and t.stride(0) < classes:
        raise ValueError(f"rows of {name} overlap")
    return rows, classes


def _refuse_scored(logits, targets):
    _on_device(logits, "logits", _TYPES)
    rows, classes = _rows(logits, "logits")
    _on_device(targets, "targets", (torch.int32, torch.int64))
    _same_device(targets, "targets", logits.device)
    if targets.shape != (rows,) or not targets.is_contiguous():
        raise ValueError(f"targets must be contiguous [{rows}], got {list(targets.shape)}")
    return rows, classes


def _refuse_log_probs(logits, targets, top):
    _, classes = _refuse_scored(logits, targets)
    if not 0 <= top <= min(_l.MAX_TOP, classes):
        raise ValueError(f"top must be between 0 and {min(_l.MAX_TOP, classes)}, got {top}")
    raise ValueError("logits cannot be used")


def _refuse_log_probs_grad(logits, targets, scored, d_logp, d_entropy, out):
    rows, _ = _refuse_scored(logits, targets)
    dev, wide = logits.device, _F64 if logits.dtype == _F64 else _F32
    if d_logp is None and d_entropy is None:
        raise ValueError("neither d_logp nor d_entropy given")
    if d_entropy is not None and scored.entropy is None:
        raise ValueError("d_entropy needs a log_probs call with want_entropy")
    for t, name, n in ((scored.stats, "stats", 4 * rows), (d_logp, "d_logp", rows), (d_entropy, "d_entropy", rows)):
        if t is not None:
            _req(t, wide, name, n)
            _same_device(t, name, dev)
    if out is not None:
        _on_device(out, "out", (logits.dtype,))
        _same_device(out, "out", dev)
        if out.shape != logits.shape:
            raise ValueError(f"out is {list(out.shape)}, the logits are {list(logits.shape)}")
        _rows(out, "out")
        raise ValueError("out overlaps the logits without being them")
    raise ValueError("logits cannot be used")


def log_probs(logits, targets, top=0, want_entropy=True):
    """Scores each row of logits [rows, classes] (fp32, fp64, bf16 or fp16; rows may be strided) at its
    target, int32 or int64 [rows], counted from 0: log probability of the target, entropy of the row,
    the `top` (at most 64) most likely classes with their log probabilities, equal logits in the order
    of their indices.  -> LogProbs; no autograd history, see log_probs_grad.  A negative target gives 0, one of `classes` or more NaN.  -inf
    logits are classes that are not allowed; a row of nothing else has log probabilities of -inf and
    entropy 0, a row with a NaN or +inf has NaN everywhere and top_index -1."""
    top = int(top)
    got = _called("log_probs", logits, logits, targets, top, bool(want_entropy))
    if got is None:
        _refuse_log_probs(logits, targets, top)
    return LogProbs(*got)


def log_probs_grad(logits, targets, scored, d_logp=None, d_entropy=None, out=None):
    """Gradient of sum(d_logp * logp) + sum(d_entropy * entropy) to the logits, from what log_probs
    returned for them.  d_logp / d_entropy: [rows] of the type of scored.logp, one of them at least.
    out: [rows, classes] of the logits' type (rows may be strided), the logits themselves allowed."""
    got = _called("log_probs_grad", logits, logits, targets, scored.stats, scored.entropy, d_logp, d_entropy, out)
    if got is None:
        _refuse_log_probs_grad(logits, targets, scored, d_logp, d_entropy, out)
    return got


def grad_norm(grads, max_norm=float("inf")):
    """Norm of the list of gradient tensors taken as one vector -> float64 [2] on their device: the norm
    and the factor min(1, max_norm / norm) that AdamW.step takes as `clip` (NaN if the norm is not
    finite: that step is then left out).  Nothing is scaled here and nothing comes back to the host."""
    grads = list(grads)
    if not grads:
        raise ValueError("grad_norm needs at least one tensor")
    max_norm = float(max_norm)
    got = _called("grad_norm", grads[0], grads, max_norm)
    if got is None:
        if not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        _refuse_list(grads, "gradient", _TYPES)
        raise ValueError("the gradients cannot be used")
    return got


class AdamW:
    """AdamW over a list of parameter tensors, all of them in one step:

        m += (1 - beta1)(g - m);  v += (1 - beta2)(g^2 - v)
        p -= lr (weight_decay p + m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps))

    params: contiguous tensors on one device (views of one flat vector as well, see param_views), fp32,
    bf16 or fp16 - or all fp64 - changed in place by step().  bf16 and fp16 parameters get an fp32
    master copy (self.master, flat in the order of the list) that takes the step; the parameter is its
    rounding, so it must not be changed from outside without load_state_dict.
    weight_decay: one factor, or one per tensor.
    state_bits=8 keeps m and sqrt(v) as e4m3 codes with one fp32 scale per 256 elements of a tensor (2.03
    bytes a parameter instead of 8; not for fp64): moments() gives the values they stand for.
    The step count lives on the device, so a captured step counts on when the graph is replayed; lr may be
    a float (kept by a captured step as it was) or a float64 [1] device tensor that is read in the step.
    Steps of one optimiser must be ordered by one stream."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter tensor")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        n = len(self.params)
        decays = [float(weight_decay)] * n if not hasattr(weight_decay, "__len__") else [float(w) for w in weight_decay]
        if len(decays) != n:
            raise ValueError(f"{len(decays)} weight_decay factors for {n} tensors")
        if not all(0 <= b < 1 for b in betas) or len(betas) != 2:
            raise ValueError(f"betas must be two numbers in [0, 1), got {betas}")
        self.device = self.params[0].device if isinstance(self.params[0], torch.Tensor) else None
        self.betas, self.eps, self.state_bits = (float(betas[0]), float(betas[1])), float(eps), state_bits
        self.lr = lr
        self._table = (_l.AdamwTensor * n)()
        first = block = 0
        spans = []
        for i, p in enumerate(self.params):
            _on_device(p, f"parameter {i}", _TYPES)
            _same_device(p, f"parameter {i}", self.device)
            if not p.is_contiguous():
                raise ValueError(f"parameter {i} must be contiguous")
            if (p.dtype == _F64) != (self.params[0].dtype == _F64):
                raise TypeError("fp64 parameters do not mix with others in one optimiser")
            if p.dtype == _F64 and state_bits == 8:
                raise TypeError("moments in 8 bits are not for fp64 parameters")
            if not (eps if p.dtype == _F64 else C.c_float(eps).value) > 0:
                raise ValueError(f"eps must be positive, in fp32 too where the parameters are not fp64, got {eps}")
            kind = _TYPES[p.dtype]
            self._table[i] = (p.data_ptr(), p.numel(), first, block, decays[i], kind)
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
            first += p.numel()
            block += -(-p.numel() // _l.MOMENT_BLOCK)
        spans.sort()
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameter tensors overlap")
        self.numel, self.blocks = first, block
        wide = _F64 if self.params[0].dtype == _F64 else _F32
        if state_bits == 32:
            self.m, self.v = (torch.zeros(first, dtype=wide, device=self.device) for _ in range(2))
            self.m_scale = self.v_scale = None
        else:
            self.m, self.v = (torch.zeros(block * _l.MOMENT_BLOCK, dtype=torch.uint8, device=self.device) for _ in range(2))
            self.m_scale, self.v_scale = (torch.zeros(block, dtype=_F32, device=self.device) for _ in range(2))
        self.master = None
        if any(p.element_size() == 2 for p in self.params):
            flat = [p.detach().reshape(-1) for p in self.params]
            same = len({p.dtype for p in self.params}) == 1
            self.master = torch.cat(flat).float() if same else torch.cat([p.float() for p in flat])
        self._clock = torch.zeros(_l.ADAMW_CLOCK, dtype=_F64, device=self.device)
        self._set_step(0)

    def _set_step(self, t):
        powers = []
        for beta in self.betas:         # multiplied step by step as the device does, so that a loaded optimiser goes on alike
            x = 1.0
            for _ in range(t):
                x, before = x * beta, x
                if x == before:         # 0, or where it stops changing
                    break
            powers.append(x)
        self._clock.copy_(torch.tensor([t, *powers] + [0.0] * (_l.ADAMW_CLOCK - 3), dtype=_F64))

    @property
    def step_count(self):
        """Steps taken so far (waits for the device)."""
        return int(self._clock[0].item())

    def step(self, grads, lr=None, clip=None):
        """One step from `grads`, one contiguous tensor per parameter with its size, of its type (or fp32
        for bf16 / fp16).  lr: instead of self.lr.  clip: grad_norm's result; its factor scales every
        gradient, and a factor that is not finite leaves everything as it is, the step count too."""
        grads, lr = list(grads), self.lr if lr is None else lr
        got = _called("adamw_step", self._clock, self.params, grads, self._table, self.state_bits, self.m, self.v,
                      self.m_scale, self.v_scale, self.master, self._clock, lr, self.betas[0], self.betas[1], self.eps, clip)
        if got is None:
            self._refuse_step(grads, lr, clip)

    def _refuse_step(self, grads, lr, clip):
        if not isinstance(self.params, list) or len(self.params) != len(self._table):
            raise ValueError(f"params must be the list of the {len(self._table)} parameters that the optimiser was made for")
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        for i, (p, t) in enumerate(zip(self.params, self._table)):
            _on_device(p, f"parameter {i}", _TYPES)
            if (p.data_ptr(), p.numel(), _TYPES[p.dtype]) != (t.param or 0, t.n, t.type):
                raise ValueError(f"parameter {i} is not what or where it was when the optimiser was made")
        _refuse_list(grads, "gradient", _TYPES)
        for i, (g, p) in enumerate(zip(grads, self.params)):
            _same_device(g, f"gradient {i}", self.device)
            if g.numel() != p.numel():
                raise ValueError(f"gradient {i} has {g.numel()} elements, its parameter {p.numel()}")
            _on_device(g, f"gradient {i}", (p.dtype, _F32) if p.element_size() == 2 else (p.dtype,))
        self._refuse_state()
        for t, name, n in ((clip, "clip", 2), (lr if isinstance(lr, torch.Tensor) else None, "lr", 1)):
            if t is not None:
                _req(t, _F64, name, n)
                _same_device(t, name, self.device)
        raise ValueError("the gradients or the optimiser's state cannot be used")

    def _refuse_state(self):
        """Raises unless the state's tensors are what the optimiser made them."""
        types, n = {t.type for t in self._table}, self.numel
        wide = _F64 if _l.TYPE_F64 in types else _F32
        want = [("m", wide, n), ("v", wide, n)]
        if self.state_bits == 8:
            codes = self.blocks * _l.MOMENT_BLOCK
            want = [("m", torch.uint8, codes), ("v", torch.uint8, codes), ("m_scale", _F32, self.blocks), ("v_scale", _F32, self.blocks)]
        if types & {_l.TYPE_BF16, _l.TYPE_F16}:
            want.append(("master", _F32, n))
        for k, dtype, size in want:
            _req(getattr(self, k), dtype, k, size)
            _same_device(getattr(self, k), k, self.device)

    def moments(self):
        """(m, v), flat in the order of the parameters: the optimiser's own tensors with 32 bits, the values
        the codes stand for (fp32) with 8."""
        if self.state_bits == 32:
            return self.m, self.v
        got = _called("adamw_moments", self.m, self._table, self.m, self.v, self.m_scale, self.v_scale, self.master)
        if got is None:
            self._refuse_state()
            raise ValueError("the optimiser's state cannot be used")
        return got

    def state_dict(self):
        """Copies of everything a later run continues from (waits for the device)."""
        keep = {k: getattr(self, k).clone() for k in ("m", "v", "m_scale", "v_scale", "master") if getattr(self, k) is not None}
        return {"step": self.step_count, **keep}

    def load_state_dict(self, state):
        """Continues from a state_dict() of an optimiser over the same tensors with the same state_bits."""
        for k in ("m", "v", "m_scale", "v_scale", "master"):
            mine, given = getattr(self, k), state.get(k)
            if (mine is None) != (given is None):
                raise ValueError(f"state {'lacks' if given is None else 'has'} {k!r}")
            if mine is not None and (mine.shape != given.shape or mine.dtype != given.dtype):
                raise ValueError(f"{k!r} is {given.dtype} {list(given.shape)}, expected {mine.dtype} {list(mine.shape)}")
        if int(state["step"]) < 0:
            raise ValueError(f"step must not be negative, got {state['step']}")
        for k in ("m", "v", "m_scale", "v_scale", "master"):
            if getattr(self, k) is not None:
                getattr(self, k).copy_(state[k])
        if self.master is not None:
            for p, t in zip(self.params, self._table):
                if p.element_size() == 2:
                    p.detach().view(-1).copy_(self.master[t.first:t.first + t.n])
        self._set_step(int(state["step"]))


def param_views(flat, z):
    """The network's six tensors W0, b0, W1, b1, W2, b2 as views of a flat parameter or gradient vector."""
    d = _l.dims(z)
    _req(flat, flat.dtype, "flat", d.nparams)
    ends = [d.off_w0, d.off_b0, d.off_w1, d.off_b1, d.off_w2, d.off_b2, d.nparams]
    return [flat[a:b] for a, b in zip(ends, ends[1:])]
