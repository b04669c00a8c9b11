"""Training operators around the pooled lookup (include/fwd_eb_train.h): the gradient of an
EmbeddingBag call, layer norm with its gradients, and AdamW over many tensors at once.

Like capi, the functions take torch CUDA tensors, launch on the current stream of the tensors'
device and return without synchronising; outputs and scratch come from torch's allocator.
Every result is deterministic; calls that accumulate into one gradient go one behind the other.
There is no CPU path.

They are the pieces of a hand-written step and stand outside autograd: results carry no graph, whatever
their inputs require.  Tensors that a call is given to write into (not AdamW's states) count as changed in place.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import os

import torch

from . import capi

BF16 = 3
BACKWARD_ACCUMULATE = 1
ADAMW_BLOCK = 256

_p, _i32, _i64 = C.c_void_p, C.c_int32, C.c_int64


class BackwardParams(C.Structure):
    """Mirror of struct fwd_eb_backward_params."""
    _fields_ = [
        ("fwd", capi.Params), ("grad_out", _p), ("grad_out_dtype", _i32), ("grad_table_dtype", _i32),
        ("grad_out_stride", _i64), ("grad_table", _p), ("grad_table_stride", _i64), ("grad_weights", _p),
        ("winners", _p), ("winners_stride", _i64), ("workspace", _p), ("workspace_bytes", C.c_size_t),
        ("flags", C.c_uint32), ("reserved", _i32),
    ]


class LayerNormParams(C.Structure):
    """Mirror of struct fwd_eb_layer_norm_params."""
    _fields_ = [
        ("x", _p), ("dtype", _i32), ("weight_dtype", _i32), ("rows", _i64), ("cols", _i64), ("x_stride", _i64),
        ("weight", _p), ("bias", _p), ("eps", C.c_double), ("mean", _p), ("rstd", _p), ("y", _p),
        ("y_stride", _i64), ("grad_y", _p), ("grad_y_stride", _i64), ("grad_x", _p), ("grad_x_stride", _i64),
        ("grad_weight", _p), ("grad_bias", _p), ("workspace", _p), ("workspace_bytes", C.c_size_t),
    ]


class AdamWTensor(C.Structure):
    """Mirror of struct fwd_eb_adamw_tensor."""
    _fields_ = [
        ("param", _p), ("grad", _p), ("master", _p), ("exp_avg", _p), ("exp_avg_sq", _p), ("exp_avg_scale", _p),
        ("exp_avg_sq_scale", _p), ("n", _i64), ("param_dtype", _i32), ("grad_dtype", _i32), ("state_bits", _i32),
        ("weight_decay", C.c_float),
    ]


class AdamWConfig(C.Structure):
    """Mirror of struct fwd_eb_adamw_config."""
    _fields_ = [
        ("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
        ("grad_scale", C.c_double), ("step", _i64), ("d_lr", _p), ("d_grad_scale", _p), ("d_step", _p),
        ("d_skip", _p),
    ]


SIGNATURES = {
    "fwd_eb_backward_params_size": (C.c_size_t, []),
    "fwd_eb_backward_workspace_size": (C.c_size_t, [_p]),
    "fwd_eb_backward": (C.c_int, [_p, _p]),
    "fwd_eb_layer_norm_params_size": (C.c_size_t, []),
    "fwd_eb_layer_norm_workspace_size": (C.c_size_t, [_p]),
    "fwd_eb_layer_norm_forward": (C.c_int, [_p, _p]),
    "fwd_eb_layer_norm_backward": (C.c_int, [_p, _p]),
    "fwd_eb_adamw_tensor_size": (C.c_size_t, []),
    "fwd_eb_adamw_config_size": (C.c_size_t, []),
    "fwd_eb_adamw_step": (C.c_int, [_p, _i32, _p, _p]),
}

_bound = None


def _lib() -> C.CDLL:
    global _bound
    if _bound is None:
        lib = capi.lib()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        for size, mirror in ((lib.fwd_eb_backward_params_size, BackwardParams),
                             (lib.fwd_eb_layer_norm_params_size, LayerNormParams),
                             (lib.fwd_eb_adamw_tensor_size, AdamWTensor),
                             (lib.fwd_eb_adamw_config_size, AdamWConfig)):
            if size() != C.sizeof(mirror):
                raise RuntimeError(f"ctypes mirror {mirror.__name__} is out of step with the library")
        _bound = lib
    return _bound


_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: BF16}


def _dtype(t, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported dtype {t.dtype}")
    return code


_OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_training_ops.so")
_loaded_ops = None


def _ops():
    """The CPython module that checks the arguments and makes the calls (csrc/torch_ops/training_ops.cpp), bound to the
    loaded library; built first if it is not there."""
    global _loaded_ops
    if _loaded_ops is None:
        if not os.path.exists(_OPS_PATH):
            from . import build as _build
            _build.build_training_ops()
        spec = importlib.util.spec_from_file_location("_training_ops", _OPS_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = _lib()
        module.bind(*(C.cast(getattr(lib, name), C.c_void_p).value for name in (
            "fwd_eb_layer_norm_forward", "fwd_eb_layer_norm_backward", "fwd_eb_layer_norm_workspace_size",
            "fwd_eb_backward", "fwd_eb_backward_workspace_size")))
        _loaded_ops = module
    return _loaded_ops


def _device_of(names, tensors) -> int:
    """Ordinal of the one CUDA device of the tensors (None ones are skipped; the first is not None)."""
    device = tensors[0].get_device()
    if device < 0:
        raise ValueError(f"{names[0]} must be a CUDA tensor; there is no CPU path")
    for name, t in zip(names, tensors):
        if t is not None and t.get_device() != device:
            if not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor; there is no CPU path")
            raise ValueError(f"{name} is on {t.device}, {names[0]} on {tensors[0].device}")
    return device


def _on(device: int, run, *args):
    """run(stream, *args) with the device current."""
    stream = (_loaded_ops or _ops()).current_stream(device, False)
    if device == torch.cuda.current_device():
        return run(stream, *args)
    with torch.cuda.device(device):
        return run(stream, *args)


# ---- gradient of the pooled lookup ----------------------------------------------------


def embedding_bag_winners(table, indices, offsets=None, *, fixed_len=0, include_last_offset=False, padding_idx=-1,
                          row_lo=0):
    """A max-pooled call that keeps what its gradient needs: fp32 pairs [num_bags, dim, 2] of the value and, as
    int32 bits, the position in the bag of the index that supplied it (FWD_EB_F32_POS).  The pooled
    rows are pairs[..., 0]; the whole tensor is embedding_bag_backward's `winners`."""
    device = _device_of(("table", "indices", "offsets"), (table, indices, offsets))
    if fixed_len == 0 and offsets is None:
        raise ValueError("offsets is None and fixed_len is 0")
    bags = indices.numel() // fixed_len if fixed_len else offsets.numel() - int(include_last_offset)

    def run(stream):
        pairs = table.new_empty((max(bags, 0), table.shape[1], 2), dtype=torch.float32)
        p = capi.make_params(table, indices, offsets, out=pairs, mode=capi.MODE_MAX, fixed_len=fixed_len,
                             include_last_offset=include_last_offset, padding_idx=padding_idx, row_lo=row_lo)
        p.out_dtype, p.out_stride = capi.F32_POS, 0
        capi.check(_lib().fwd_eb_forward(C.byref(p), stream))
        return pairs
    return _on(device, run)


def embedding_bag_backward(grad_out, table, indices, offsets=None, *, mode=capi.MODE_SUM, fixed_len=0,
                           per_sample_weights=None, include_last_offset=False, padding_idx=-1, row_lo=0, flags=0,
                           winners=None, grad_table=None, grad_dtype=None, accumulate=False, need_table=True,
                           need_weights=False):
    """Gradients of capi.embedding_bag(table, indices, offsets, ...) for grad_out = d loss / d out.

    Returns (grad_table, grad_weights).  grad_table is dense, [num_rows, dim] over the table's rows, in
    `grad_dtype` (default: the table's) or the tensor given as `grad_table`; with accumulate=True
    the gradient is added to what that tensor holds, at a cost that goes by the lookups and not by the
    table.  grad_weights is fp32, [num_indices].  What is not asked for is None.  MODE_MAX takes
    `winners` from embedding_bag_winners.
    """
    result = (_loaded_ops or _ops()).embedding_bag_backward(
        grad_out, table, indices, offsets, mode, fixed_len, per_sample_weights, include_last_offset, padding_idx, row_lo,
        flags, winners, grad_table, _asked(grad_dtype, "grad_dtype"), accumulate, need_table, need_weights)
    if type(result) is int:
        capi.check(result)
    return result


def _asked(dtype, what: str) -> int:
    """The code of a dtype that was asked for, -1 for None."""
    if dtype is None:
        return -1
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    return _DTYPES[dtype]


# ---- layer norm -------------------------------------------------------------------------


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None, return_stats=False):
    """Layer norm of the rows of x [rows, cols] (fp32, fp16 or bf16; any row stride).

    Returns y of x's dtype (`out`, which may be x, or a new tensor), or (y, mean, rstd) with
    return_stats=True: the fp32 statistics that layer_norm_backward takes."""
    result = (_loaded_ops or _ops()).layer_norm(x, weight, bias, eps, out, return_stats)
    if type(result) is int:
        capi.check(result)
    return result


def layer_norm_backward(grad_y, x, mean, rstd, weight=None, *, grad_x=None, need_x=True, need_params=True,
                        param_dtype=None):
    """Gradients of layer_norm: (grad_x, grad_weight, grad_bias).

    mean and rstd are the forward call's.  grad_x (x's dtype) may be given, and may be grad_y or x
    itself.  grad_weight and grad_bias have the weight's dtype, or `param_dtype` (default fp32)
    where there is no weight.  What is not asked for is None."""
    result = (_loaded_ops or _ops()).layer_norm_backward(grad_y, x, mean, rstd, weight, grad_x, need_x, need_params,
                                                         _asked(param_dtype, "param_dtype"))
    if type(result) is int:
        capi.check(result)
    return result


# ---- AdamW ------------------------------------------------------------------------------


class AdamW:
    """AdamW over a list of contiguous CUDA tensors of one device, one launch a step (per 256 tensors).

    state_bits=32 keeps exp_avg and exp_avg_sq in fp32; 8 keeps exp_avg and the square root of
    exp_avg_sq as float8_e4m3fn with one fp32 scale per 256 elements (exp_avg_scale,
    exp_avg_sq_scale): the value of element i is float(code[i]) * scale[i // 256].  masters[i], fp32, is
    the copy that the step works on where parameter i is fp16 or bf16; the parameter is then
    its rounded image.  The state tensors may be given (to resume); otherwise they start at zero.
    weight_decay is a number, or one per tensor.  The optimizer addresses the tensors' memory: a tensor that
    is given other memory (p.data = ...) needs a new one.

    capturable=True keeps the step count and lr on the device (step_tensor, lr_tensor): a step
    captured into a graph then counts on with every replay, and lr may be changed in between.
    """

    def __init__(self, params, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 masters=None, exp_avg=None, exp_avg_sq=None, exp_avg_scale=None, exp_avg_sq_scale=None, step=0,
                 capturable=False):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits is 32 or 8 (got {state_bits})")
        self._ordinal = _device_of([f"params[{i}]" for i in range(len(self.params))], self.params)
        self.device = self.params[0].device
        self.state_bits = state_bits
        self.step_count = int(step)
        if self.step_count < 0:
            raise ValueError(f"step counts the steps that were made (got {step})")
        n = len(self.params)
        decay = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(d) for d in weight_decay]
        if len(decay) != n:
            raise ValueError("weight_decay: one number, or one per parameter")
        state = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        blocks = [-(-p.numel() // ADAMW_BLOCK) for p in self.params]
        if state_bits == 32 and (exp_avg_scale is not None or exp_avg_sq_scale is not None):
            raise ValueError("states of 32 bits have no scales")

        def states(given, name, dtype, sizes):
            if given is None:
                return [torch.zeros(k, dtype=dtype, device=self.device) for k in sizes]
            given = list(given)
            if len(given) != n:
                raise ValueError(f"{name}: one tensor per parameter")
            for i, t in enumerate(given):
                self._check(t, f"{name}[{i}]", sizes[i])
                if t.dtype != dtype:
                    raise TypeError(f"{name}[{i}] must be {dtype}")
            return given

        for i, p in enumerate(self.params):
            self._check(p, f"params[{i}]", p.numel())
            _dtype(p, f"params[{i}]")
        sizes = [p.numel() for p in self.params]
        self.masters = [None] * n if masters is None else list(masters)
        if len(self.masters) != n:
            raise ValueError("masters: one tensor (or None) per parameter")
        for i, t in enumerate(self.masters):
            if t is not None:
                self._check(t, f"masters[{i}]", sizes[i])
                if t.dtype != torch.float32:
                    raise TypeError(f"masters[{i}] must be fp32")
        self.exp_avg = states(exp_avg, "exp_avg", state, sizes)
        self.exp_avg_sq = states(exp_avg_sq, "exp_avg_sq", state, sizes)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale = states(exp_avg_scale, "exp_avg_scale", torch.float32, blocks)
            self.exp_avg_sq_scale = states(exp_avg_sq_scale, "exp_avg_sq_scale", torch.float32, blocks)
        written = self.params + [t for t in self.masters if t is not None] + self.exp_avg + self.exp_avg_sq
        written += (self.exp_avg_scale or []) + (self.exp_avg_sq_scale or [])
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in written if t.numel())
        if any(end > begin for (_, end), (begin, _) in zip(spans, spans[1:])):
            raise ValueError("a parameter, master copy or state is there twice, or two of them overlap")
        self._valued = self.params + [t for t in self.masters if t is not None]     # what a loss may have been computed from
        self._table = (AdamWTensor * n)()
        for i, p in enumerate(self.params):
            t = self._table[i]
            t.param, t.n, t.param_dtype = p.data_ptr(), p.numel(), _DTYPES[p.dtype]
            t.master = None if self.masters[i] is None else self.masters[i].data_ptr()
            t.exp_avg, t.exp_avg_sq = self.exp_avg[i].data_ptr(), self.exp_avg_sq[i].data_ptr()
            if state_bits == 8:
                t.exp_avg_scale = self.exp_avg_scale[i].data_ptr()
                t.exp_avg_sq_scale = self.exp_avg_sq_scale[i].data_ptr()
            t.state_bits, t.weight_decay = state_bits, decay[i]
        self._config = AdamWConfig(lr, betas[0], betas[1], eps, 1.0, 0, None, None, None, None)
        self.step_tensor = self.lr_tensor = None
        if capturable:
            self.step_tensor = torch.full((1,), self.step_count, dtype=torch.int64, device=self.device)
            self.lr_tensor = torch.full((1,), lr, dtype=torch.float32, device=self.device)
            self._config.d_step, self._config.d_lr = self.step_tensor.data_ptr(), self.lr_tensor.data_ptr()
        self._config_ref = C.byref(self._config)
        self._host = AdamWConfig(lr, betas[0], betas[1], eps, 1.0, 1, None, None, None, None)   # see step
        self._grads = None
        self._captured = []         # what captured steps read beside gradients and states
        self._lib = _lib()
        self._config.step = 1
        capi.check(self._lib.fwd_eb_adamw_step(None, 0, self._config_ref, None))   # refuses what is out of range

    def _check(self, t, name, numel):
        if not t.is_cuda or t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        if t.numel() != numel or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous, {numel} elements")

    def bind(self, grads) -> None:
        """Gradients of the steps to come, one per parameter: buffers that the caller refills between steps.
        They are kept alive until the next bind."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError("one gradient per parameter")
        for i, g in enumerate(grads):
            self._check(g, f"grads[{i}]", self._table[i].n)
            _dtype(g, f"grads[{i}]")
        for t, g in zip(self._table, grads):
            t.grad, t.grad_dtype = g.data_ptr(), _DTYPES[g.dtype]
        self._grads = grads

    def step(self, grads=None, *, lr=None, grad_scale=1.0, skip=None) -> None:
        """One step with `grads` (bound first) or the bound gradients.  lr, where given, holds from this step
        on.  grad_scale: a number, or an fp32 device tensor of one element.  skip: an int32
        device tensor of one element; where it is not 0 the step changes nothing (it still counts).
        A capture into a graph wants capturable=True: the numbers of any other step are the graph's for good.  The
        graph reads the tensors of the captured call: the optimizer keeps grad_scale and skip alive as long as it lives
        itself; it and the gradients have to outlive the graph."""
        if grads is not None:
            self.bind(grads)
        if self._grads is None:
            raise ValueError("no gradients: give them here or call bind()")
        cfg = self._config
        for name, t, dtype in (("grad_scale", grad_scale, torch.float32), ("skip", skip, torch.int32)):
            if isinstance(t, torch.Tensor):
                self._check(t, name, 1)
                if t.dtype != dtype:
                    raise TypeError(f"{name} must be {dtype}")
        if skip is not None and not isinstance(skip, torch.Tensor):
            raise TypeError("skip must be an int32 device tensor")
        if isinstance(grad_scale, torch.Tensor):
            cfg.d_grad_scale = grad_scale.data_ptr()
        else:
            cfg.d_grad_scale, cfg.grad_scale = None, grad_scale
        cfg.d_skip = None if skip is None else skip.data_ptr()
        scalars = [t for t in (grad_scale, skip) if isinstance(t, torch.Tensor)]
        if self.step_tensor is not None:      # what the call would refuse is refused before the device's numbers move
            self._host.grad_scale = 1.0 if cfg.d_grad_scale else grad_scale
            if lr is not None and not isinstance(lr, torch.Tensor):
                self._host.lr = lr
            try:
                capi.check(self._lib.fwd_eb_adamw_step(None, 0, C.byref(self._host), None))
            finally:
                self._host.lr = cfg.lr
        before = cfg.lr
        if self.step_tensor is None:
            if lr is not None:
                cfg.lr = lr
            cfg.step = self.step_count + 1
        try:
            stream = (_loaded_ops or _ops()).current_stream(self._ordinal, self.step_tensor is None)
            if self._ordinal == torch.cuda.current_device():
                self._launch(stream, lr, scalars)
            else:
                with torch.cuda.device(self._ordinal):
                    self._launch(stream, lr, scalars)
        except Exception:
            cfg.lr = before
            raise
        self.step_count += 1
        _loaded_ops.touched(self._valued)

    def _launch(self, stream, lr, scalars):
        if self.step_tensor is not None:
            if scalars and torch.cuda.is_current_stream_capturing():
                self._captured += scalars
            if lr is not None:
                self.lr_tensor.fill_(lr)
            self.step_tensor.add_(1)
        capi.check(self._lib.fwd_eb_adamw_step(self._table, len(self._table), self._config_ref, stream))
