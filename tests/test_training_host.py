"""CPU-side checks of the training operators: struct mirrors, exported symbols, argument errors that are
reported before any launch, workspace sizes, and the Python layer's own refusals."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from forward_b200 import capi, training as T  # noqa: E402


def _lib():
    return T._lib()


def _back(**kw):
    f = capi.Params(0x1000, capi.F16, 128, 1000, 0, 0, 0x2000, 0x3000, capi.I32, 0, 4000, 100, None, capi.MODE_SUM,
                    0, -1, None, 0, 0, 0, None, 0, 0, 0)
    p = T.BackwardParams()
    for k in list(kw):
        if k.startswith("fwd_"):
            setattr(f, k[4:], kw.pop(k))
    p.fwd = f
    p.grad_out, p.grad_out_dtype, p.grad_table_dtype = 0x10000, capi.F16, capi.F16
    p.grad_table, p.workspace, p.workspace_bytes = 0x20000, 0x100000, 1 << 40
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _norm(backward, **kw):
    p = T.LayerNormParams(0x1000, capi.F16, capi.F32, 100, 64, 0, 0x2000, 0x3000, 1e-5, 0x4000, 0x5000)
    if backward:
        p.grad_y, p.grad_x, p.grad_weight, p.grad_bias = 0x6000, 0x7000, 0x8000, 0x9000
        p.workspace, p.workspace_bytes = 0x100000, 1 << 40
    else:
        p.y = 0x6000
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _tensor(**kw):
    t = T.AdamWTensor(0x1000, 0x2000, None, 0x3000, 0x4000, None, None, 1000, capi.F32, capi.F32, 32, 0.01)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _config(**kw):
    c = T.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 1.0, 1, None, None, None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _refused(rc, code, before):
    assert rc == code
    assert _lib().fwd_eb_last_error_string() != b""
    assert _lib().fwd_eb_launch_count() == before


def test_struct_mirrors():
    lib = _lib()
    assert lib.fwd_eb_backward_params_size() == C.sizeof(T.BackwardParams)
    assert lib.fwd_eb_layer_norm_params_size() == C.sizeof(T.LayerNormParams)
    assert lib.fwd_eb_adamw_tensor_size() == C.sizeof(T.AdamWTensor) == 80
    assert lib.fwd_eb_adamw_config_size() == C.sizeof(T.AdamWConfig)


@pytest.mark.parametrize("kw,code", [
    (dict(grad_out=None), capi.EINVAL),
    (dict(grad_out_dtype=T.BF16), capi.EINVAL),
    (dict(grad_table_dtype=7), capi.EINVAL),
    (dict(grad_table=None), capi.EINVAL),
    (dict(grad_out_stride=64), capi.EINVAL),
    (dict(grad_table_stride=127), capi.EINVAL),
    (dict(flags=2), capi.EINVAL),
    (dict(fwd_mode=capi.MODE_MAX), capi.EINVAL),                          # no winners
    (dict(fwd_mode=capi.MODE_MAX, winners=0x40004), capi.EALIGN),
    (dict(fwd_mode=capi.MODE_MAX, winners=0x40000, winners_stride=100), capi.EINVAL),
    (dict(fwd_mode=capi.MODE_MEAN, grad_weights=0x50000), capi.EINVAL),
    (dict(fwd_mode=capi.MODE_SQUARE_SUM, fwd_table=None), capi.EINVAL),
    (dict(fwd_table=None, grad_weights=0x50000), capi.EINVAL),
    (dict(fwd_mode=capi.MODE_MEAN, fwd_per_sample_weights=0x60000), capi.EINVAL),
    (dict(fwd_flags=capi.FLAG_OFFSET_PAIRS), capi.EUNSUPPORTED),
    (dict(fwd_num_indices=2**31 - 1), capi.ETOOBIG),
    (dict(fwd_num_rows=2**31), capi.ETOOBIG),
    (dict(fwd_dim=2**20 + 1), capi.ETOOBIG),
    (dict(fwd_offsets=None), capi.EINVAL),
    (dict(fwd_fixed_len=7), capi.EINVAL),
    (dict(grad_out=0x10001), capi.EALIGN),
    (dict(fwd_indices=0x2002), capi.EALIGN),
    (dict(workspace_bytes=1000), capi.EWORKSPACE),
    (dict(workspace=None), capi.EWORKSPACE),
    (dict(workspace=0x100010), capi.EALIGN),
])
def test_backward_refusals(kw, code):
    before = _lib().fwd_eb_launch_count()
    p = _back(**kw)
    _refused(_lib().fwd_eb_backward(C.byref(p), None), code, before)


def test_backward_workspace():
    lib = _lib()
    need = lib.fwd_eb_backward_workspace_size(C.byref(_back()))
    n, dim = 4000, 128
    runs = n // 32
    assert need >= n * 16 + runs * 2 * dim * 4
    assert lib.fwd_eb_backward_workspace_size(C.byref(_back(grad_table=None, grad_weights=0x50000))) < need
    assert lib.fwd_eb_backward_workspace_size(C.byref(_back(fwd_num_indices=0))) == 0
    assert lib.fwd_eb_backward_workspace_size(C.byref(_back(fwd_mode=77))) == 0
    assert lib.fwd_eb_backward(None, None) == capi.EINVAL
    # padding makes a mean count, which takes one word a bag
    mean = lib.fwd_eb_backward_workspace_size(C.byref(_back(fwd_mode=capi.MODE_MEAN)))
    assert lib.fwd_eb_backward_workspace_size(C.byref(_back(fwd_mode=capi.MODE_MEAN, fwd_padding_idx=0))) > mean


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(x=None), capi.EINVAL),
    (dict(dtype=2), capi.EINVAL),
    (dict(weight_dtype=9), capi.EINVAL),
    (dict(rows=-1), capi.EINVAL),
    (dict(cols=0), capi.EINVAL),
    (dict(cols=2**30 + 1), capi.ETOOBIG),
    (dict(x_stride=63), capi.EINVAL),
    (dict(x=0x1001), capi.EALIGN),
    (dict(weight=0x2002), capi.EALIGN),
    (dict(mean=0x4001), capi.EALIGN),
])
def test_layer_norm_refusals(backward, kw, code):
    before = _lib().fwd_eb_launch_count()
    fn = _lib().fwd_eb_layer_norm_backward if backward else _lib().fwd_eb_layer_norm_forward
    _refused(fn(C.byref(_norm(backward, **kw)), None), code, before)


@pytest.mark.parametrize("backward,kw,code", [
    (False, dict(y=None), capi.EINVAL),
    (False, dict(y_stride=10), capi.EINVAL),
    (False, dict(eps=-1e-5), capi.EINVAL),
    (False, dict(eps=float("nan")), capi.EINVAL),
    (True, dict(grad_y=None), capi.EINVAL),
    (True, dict(mean=None), capi.EINVAL),
    (True, dict(rstd=None), capi.EINVAL),
    (True, dict(grad_x_stride=8), capi.EINVAL),
    (True, dict(grad_bias=0x9002), capi.EALIGN),
    (True, dict(workspace_bytes=100), capi.EWORKSPACE),
    (True, dict(workspace=0x100080), capi.EALIGN),
])
def test_layer_norm_refusals_of_one_direction(backward, kw, code):
    before = _lib().fwd_eb_launch_count()
    fn = _lib().fwd_eb_layer_norm_backward if backward else _lib().fwd_eb_layer_norm_forward
    _refused(fn(C.byref(_norm(backward, **kw)), None), code, before)


def test_layer_norm_workspace_and_empty():
    lib = _lib()
    assert lib.fwd_eb_layer_norm_workspace_size(C.byref(_norm(True))) >= 2 * 64 * 4
    assert lib.fwd_eb_layer_norm_workspace_size(C.byref(_norm(True, grad_weight=None, grad_bias=None))) == 0
    assert lib.fwd_eb_layer_norm_workspace_size(C.byref(_norm(True, rows=0))) == 0
    assert lib.fwd_eb_layer_norm_workspace_size(None) == 0
    assert lib.fwd_eb_layer_norm_forward(None, None) == capi.EINVAL
    assert lib.fwd_eb_layer_norm_backward(None, None) == capi.EINVAL
    before = lib.fwd_eb_launch_count()
    assert lib.fwd_eb_layer_norm_forward(C.byref(_norm(False, rows=0, x=None, y=None)), None) == 0
    assert lib.fwd_eb_launch_count() == before


@pytest.mark.parametrize("tkw,ckw,code", [
    (dict(param=None), {}, capi.EINVAL),
    (dict(grad=None), {}, capi.EINVAL),
    (dict(exp_avg=None), {}, capi.EINVAL),
    (dict(n=-1), {}, capi.EINVAL),
    (dict(n=2**41), {}, capi.ETOOBIG),
    (dict(param_dtype=2), {}, capi.EINVAL),
    (dict(grad_dtype=4), {}, capi.EINVAL),
    (dict(state_bits=16), {}, capi.EINVAL),
    (dict(state_bits=8), {}, capi.EINVAL),                                # no scales
    (dict(exp_avg_scale=0x5000), {}, capi.EINVAL),                        # scales of 32-bit states
    (dict(weight_decay=float("inf")), {}, capi.EINVAL),
    (dict(param=0x1002), {}, capi.EALIGN),
    (dict(master=0x1001), {}, capi.EALIGN),
    ({}, dict(lr=-1.0), capi.EINVAL),
    ({}, dict(lr=float("nan")), capi.EINVAL),
    ({}, dict(beta1=1.0), capi.EINVAL),
    ({}, dict(beta2=-0.1), capi.EINVAL),
    ({}, dict(eps=float("inf")), capi.EINVAL),
    ({}, dict(step=0), capi.EINVAL),
    ({}, dict(grad_scale=float("nan")), capi.EINVAL),
    ({}, dict(d_step=0x1004), capi.EALIGN),
])
def test_adamw_refusals(tkw, ckw, code):
    before = _lib().fwd_eb_launch_count()
    ts = (T.AdamWTensor * 2)(_tensor(), _tensor(**tkw))   # the second is bad: nothing may run
    _refused(_lib().fwd_eb_adamw_step(ts, 2, C.byref(_config(**ckw)), None), code, before)


def test_adamw_empty_lists():
    lib = _lib()
    assert lib.fwd_eb_adamw_step(None, 0, C.byref(_config()), None) == 0
    assert lib.fwd_eb_adamw_step(None, 1, C.byref(_config()), None) == capi.EINVAL
    assert lib.fwd_eb_adamw_step(None, -1, C.byref(_config()), None) == capi.EINVAL
    ts = (T.AdamWTensor * 1)(_tensor(n=0, param=None, grad=None))
    assert lib.fwd_eb_adamw_step(ts, 1, None, None) == capi.EINVAL
    before = lib.fwd_eb_launch_count()
    assert lib.fwd_eb_adamw_step(ts, 1, C.byref(_config()), None) == 0
    assert lib.fwd_eb_launch_count() == before


def test_python_layer_takes_cuda_tensors_only():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="no CPU path"):
        T.layer_norm(x)
    with pytest.raises(ValueError, match="no CPU path"):
        T.layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="no CPU path"):
        T.embedding_bag_backward(x, x, torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="no CPU path"):
        T.AdamW([x])
    with pytest.raises(ValueError):
        T.AdamW([])
