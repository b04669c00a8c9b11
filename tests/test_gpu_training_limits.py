"""The training operators at the edges of what their calls allow, on the GPU against plain 64-bit forms: values
next to fp32's smallest, constant rows, chains of calls on one stream, refused and captured steps.

Tolerances are bounds of the arithmetic, as in test_gpu_training.py, whose helpers are used.
"""
import ctypes as C
import gc
import math
import weakref

import pytest

torch = pytest.importorskip("torch")

from forward_b200 import capi, training as T  # noqa: E402
from test_gpu_training import DEV, F64, HYPER, U, adam_case, from_codes, gen, make_bags, same_bits, within  # noqa: E402

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -149       # the smallest fp32 value; a result below 2^-126 is off by at most half of it


# ---- AdamW: gradients whose squares leave fp32's normal range -------------------------------


def faint(n, seed):
    """Magnitudes of 3e-20 to 3e-18, evenly over the logarithm: 0.05 g^2 lies on both sides of 2^-126."""
    g = gen(seed)
    size = 10.0 ** (torch.rand(n, generator=g, device=DEV, dtype=F64) * 2 - 19.5)
    sign = torch.randint(0, 2, (n,), generator=g, device=DEV) * 2 - 1
    return (size * sign).float()


def check_faint_step(opt, g, step, hyper):
    """One step of one fp32 tensor, against the update in 64 bits from the states as they are held before it."""
    lr, (b1, b2), eps, wd = hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"]
    p = opt.params[0].to(F64)
    if opt.state_bits == 8:
        m, root = from_codes(opt.exp_avg[0], opt.exp_avg_scale[0]), from_codes(opt.exp_avg_sq[0], opt.exp_avg_sq_scale[0])
        v = root.square()
    else:
        m, v = opt.exp_avg[0].to(F64), opt.exp_avg_sq[0].to(F64)
    opt.step([g])
    g = g.to(F64)
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    root = v1.sqrt()
    correct = 1 / math.sqrt(1 - b2 ** step)
    den = root * correct + eps
    upd = lr / (1 - b1 ** step) * m1 / den
    # m: as for any gradient.  v: ten roundings, and at most six products and sums that may fall below 2^-126
    dm = 8 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 4 * LEAST
    dv = 10 * U * v1 + 3 * LEAST
    # |sqrt(a) - sqrt(b)| <= |a - b| / sqrt(b); 2^-24 more where eps may hide a v below 2^-126
    dden = dv / root * correct + U * eps
    bound = upd.abs() * (16 * U + dden / (den - dden)) + lr / (1 - b1 ** step) * dm / (den - dden)
    within(opt.params[0], p * (1 - lr * wd) - upd, bound + 4 * U * (p.abs() + upd.abs()), "param")


@pytest.mark.parametrize("eps", [1e-25, 1e-20, 1e-17, 1e-13, 1.7e-11, 1e-8])
@pytest.mark.parametrize("n", [5000, 9_000_001])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_first_step_from_faint_gradients(bits, n, eps):
    """Short chunks and, with 8-bit states, the long ones whose loads are under way together: one formula for both, for
    an eps below, among and above the roots of the smallest v."""
    hyper = dict(HYPER, eps=eps)
    opt = T.AdamW([torch.randn(n, generator=gen(n), device=DEV)], state_bits=bits, **hyper)
    check_faint_step(opt, faint(n, 1), 1, hyper)


@pytest.mark.parametrize("n,eps", [(5000, 1e-20), (5000, 1e-8), (9_000_001, 1e-20), (9_000_001, 1.7e-11)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps_from_faint_states(bits, n, eps):
    """Later steps, from states that faint gradients left: what 8 bits hold is taken at its value, though its
    scale's square is below 2^-126."""
    hyper = dict(HYPER, eps=eps)
    opt = T.AdamW([torch.randn(n, generator=gen(n), device=DEV)], state_bits=bits, **hyper)
    opt.step([faint(n, 1)])
    for step in (2, 3):
        check_faint_step(opt, faint(n, step), step, hyper)


# ---- calls one behind the other ------------------------------------------------------------------


@pytest.mark.parametrize("lengths", [[8] * 40, [40] * 2000, [300] * 60])
def test_max_gradient_right_behind_its_forward_call(lengths):
    """The winners are read while the launches of the call that wrote them may still be the ones ahead: every batch anew
    into the same memory, the results of a run that waits after each call."""
    batches = [make_bags(seed, 900, 64, lengths, mode=capi.MODE_MAX, dtype=torch.float32) for seed in range(6)]
    pairs = torch.empty(len(lengths), 64, 2, device=DEV)

    def run(wait):
        got = []
        for s, go, _, _ in batches * 3:
            p = capi.make_params(s["table"], s["indices"], s["offsets"], out=pairs, mode=capi.MODE_MAX)
            p.out_dtype, p.out_stride = capi.F32_POS, 0
            capi.forward(p)
            wait()
            got.append(T.embedding_bag_backward(go, s["table"], s["indices"], s["offsets"], mode=capi.MODE_MAX, winners=pairs)[0])
            wait()
        return got

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bags,rows", [(16, 200), (3000, 20_000)])
def test_steps_and_lookups_right_behind_one_another(bags, rows, bits):
    """The table that a step writes is pooled by the next call on the stream, its gradient taken, and so on, per-sample
    weights among the parameters: the bits of a loop that waits after each call."""
    batches = [make_bags(seed, rows, 64, [9] * bags, mode=capi.MODE_SUM, dtype=torch.float32) for seed in range(4)]

    def run(wait):
        table, w = torch.randn(rows, 64, generator=gen(1), device=DEV), torch.rand(9 * bags, generator=gen(2), device=DEV)
        grad, gw = torch.empty_like(table), torch.empty_like(w)
        opt = T.AdamW([table, w], state_bits=bits, **HYPER)
        opt.bind([grad, gw])
        kept = []
        for s, go, _, _ in batches * 4:
            pooled = capi.embedding_bag(table, s["indices"], s["offsets"], per_sample_weights=w)
            wait()
            y, mean, rstd = T.layer_norm(pooled, return_stats=True)
            wait()
            rows_again = capi.embedding_bag(y, s["indices"][:8] % bags, mode=capi.MODE_GATHER)     # the norm's rows as a table
            wait()
            gx, _, _ = T.layer_norm_backward(go, pooled, mean, rstd)
            wait()
            _, dw = T.embedding_bag_backward(gx, table, s["indices"], s["offsets"], per_sample_weights=w, grad_table=grad,
                                             need_weights=True)
            wait()
            again = capi.embedding_bag(grad, s["indices"], s["offsets"], per_sample_weights=dw)      # gradients as inputs
            wait()
            gw.copy_(dw)
            opt.step()
            wait()
            kept += [pooled, rows_again, again]
        return kept + [table, w]

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, want))


# ---- refused and captured steps --------------------------------------------------------------------


@pytest.mark.parametrize("kw", [dict(grad_scale=float("inf")), dict(grad_scale=1e39), dict(lr=-1.0), dict(lr=float("nan")),
                                dict(lr=0.5, grad_scale=float("nan"))])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_leaves_the_optimizer_as_it_was(capturable, kw):
    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    opt = T.AdamW([p], lr=0.25, capturable=capturable)
    opt.step([g])
    before = [t.clone() for t in (p, *opt.exp_avg, *opt.exp_avg_sq)]
    for _ in range(2):
        with pytest.raises(capi.FwdEbError):
            opt.step([g], **kw)
    assert all(same_bits(a, b) for a, b in zip(before, (p, *opt.exp_avg, *opt.exp_avg_sq)))
    assert opt.step_count == 1
    if capturable:
        assert int(opt.step_tensor) == 1 and float(opt.lr_tensor) == 0.25
    opt.step([g], lr=0.125)                                  # from the lr and the count of before
    other = torch.ones(300, device=DEV)
    plain = T.AdamW([other], lr=0.25, capturable=capturable)
    plain.step([g])
    plain.step([g], lr=0.125)
    assert same_bits(p, other)
    assert not capturable or (int(opt.step_tensor) == 2 and float(opt.lr_tensor) == 0.125)


def test_a_captured_step_keeps_its_scale_and_skip_flag():
    """Made for the call and dropped by the caller: their memory stays theirs, and each replay reads what they held."""
    p, g = torch.zeros(300, device=DEV), torch.ones(300, device=DEV)
    opt = T.AdamW([p], lr=0.25, betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, capturable=True)
    opt.bind([g])
    scale, skip = torch.full((1,), 3.0, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    held = [weakref.ref(scale), weakref.ref(skip)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grad_scale=scale, skip=skip)
    del scale, skip
    gc.collect()
    assert all(r() is not None for r in held)
    filler = [torch.full((1,), -7, dtype=torch.int32, device=DEV) for _ in range(200)]     # what freed memory would turn into
    graph.replay()
    # m = 3, v = 9: a step of lr * 3 / (3 + 1)
    assert torch.equal(p, torch.full_like(p, -0.25 * 3 / 4)) and len(filler) == 200
    eager = torch.full((1,), 3.0, device=DEV)
    opt.step(grad_scale=eager)
    held = weakref.ref(eager)
    del eager
    assert held() is None                                    # nobody replays an eager step


# ---- autograd's bookkeeping ------------------------------------------------------------------------


def test_tensors_written_in_place_count_as_changed():
    """Autograd refuses to differentiate through a saved tensor that a call has overwritten; what was only read does not count."""
    x, w = torch.randn(20, 16, device=DEV), torch.ones(16, device=DEV)
    g, stats = torch.randn(20, 16, device=DEV), T.layer_norm(x, return_stats=True)[1:]
    idx, off = torch.zeros(40, dtype=torch.int32, device=DEV), torch.arange(0, 40, 2, dtype=torch.int32, device=DEV)

    def writes(out, call, *read):
        before = out._version, [t._version for t in read]
        leaf = torch.ones_like(out, requires_grad=True)
        loss = (leaf * out).sum()
        call()
        assert out._version == before[0] + 1 and [t._version for t in read] == before[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

    for out in (torch.empty_like(x), x.clone()):
        writes(out, lambda: T.layer_norm(x, w, out=out), x, w)
        writes(out, lambda: T.layer_norm_backward(g, x, *stats, w, grad_x=out), g, x, w, *stats)
    for rows in (30, 5000):
        table, grad = torch.randn(rows, 16, device=DEV), torch.zeros(rows, 16, device=DEV)
        for accumulate in (False, True):
            writes(grad, lambda: T.embedding_bag_backward(g, table, idx, off, grad_table=grad, accumulate=accumulate), g, table, idx)
    T.layer_norm(x, w)
    assert x._version == 0
    for bits in (32, 8):
        p, master = torch.ones(300, device=DEV).half(), torch.ones(300, device=DEV)
        opt = T.AdamW([p], masters=[master], state_bits=bits)
        grad = torch.ones(300, device=DEV)
        for t in (p, master):
            before = t._version
            opt.step([grad])
            assert t._version == before + 1
        assert grad._version == 0
    p = torch.ones(300, device=DEV, requires_grad=True)
    loss = (p * p).sum()
    T.AdamW([p]).step([torch.ones(300, device=DEV)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_of_inference_mode_are_taken():
    with torch.inference_mode():
        x, p = torch.randn(20, 16, device=DEV), torch.ones(300, device=DEV)
        opt = T.AdamW([p])
    T.layer_norm(x, out=x)
    opt.step([torch.ones(300, device=DEV)])
    assert (p < 1).all() and abs(float(x.mean())) < 1e-5


def test_results_stand_outside_autograd():
    x = torch.randn(20, 16, device=DEV, requires_grad=True)
    y, mean, rstd = T.layer_norm(x, return_stats=True)
    assert not y.requires_grad and not T.layer_norm_backward(y, x, mean, rstd)[0].requires_grad


# ---- layer norm: rows of one value ------------------------------------------------------------------


@pytest.mark.parametrize("cols", [7, 41, 60, 63, 95, 100, 250, 777, 1000, 1023, 2000, 4095, 5000, 8000, 8191, 9000, 16000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layer_norm_of_constant_rows_of_any_width(dtype, cols):
    """x - mean is 0 in a row of one value, so y is the bias, and a constant grad_y has no gradient.  The values are small
    integers: every sum of them is exact in fp32 (below 2^24), and so is the quotient."""
    values = [1.0, 3.0, -7.0, 100.0, 1000.0]        # of 8 bits at most: bf16 holds them (1000 = 125 * 8)
    x = torch.tensor(values, device=DEV).to(dtype)[:, None].expand(-1, cols).contiguous()
    bias = torch.randn(cols, generator=gen(cols), device=DEV)
    y, mean, rstd = T.layer_norm(x, None, bias, return_stats=True)
    assert mean.tolist() == values
    assert torch.equal(y, bias.to(dtype).expand(len(values), -1))
    # h = 0 and g - mean(g) = 0
    gx, gw, gb = T.layer_norm_backward(x, x, mean, rstd)
    assert not gx.any() and not gw.any() and torch.equal(gb, torch.full_like(gb, sum(values)))


@pytest.mark.parametrize("cols", [100, 1000, 20000])
def test_layer_norm_mean_of_an_infinite_row(cols):
    x = torch.ones(3, cols, device=DEV)
    x[1, 5] = float("inf")
    y, mean, _ = T.layer_norm(x, return_stats=True)
    assert mean.tolist() == [1.0, float("inf"), 1.0]
    assert torch.isnan(y[1, 5]) and not y[[0, 2]].any()


# ---- what AdamW is made from ----------------------------------------------------------------------


def test_adamw_refuses_tensors_that_overlap():
    """Every tensor of a step is a thread's own to read and write: views that share a part are as wrong as the same one twice."""
    flat, state = torch.zeros(1000, device=DEV), torch.zeros(1000, device=DEV)
    for a, b in ((flat[:600], flat[599:]), (flat[100:200], flat), (flat[600:], flat[:601])):
        with pytest.raises(ValueError, match="overlap"):
            T.AdamW([a, b])
    with pytest.raises(ValueError, match="overlap"):
        T.AdamW([flat[:500]], exp_avg=[state[:500]], exp_avg_sq=[state[499:999]])
    with pytest.raises(ValueError, match="overlap"):
        T.AdamW([flat[:500].view(torch.float16)], masters=[torch.zeros(1000, device=DEV)], exp_avg=[flat[499:1000].new_zeros(1000)],
                exp_avg_sq=[flat])
    halves = T.AdamW([flat[:500], flat[500:], flat[3:3]], exp_avg=[state[500:], state[:500], state[:0]])
    halves.step([torch.ones(500, device=DEV), torch.ones(500, device=DEV), torch.zeros(0, device=DEV)])
    assert (flat < 0).all() and same_bits(flat[:500], flat[500:])


@pytest.mark.parametrize("capturable", [False, True])
def test_adamw_refuses_a_negative_step_count(capturable):
    """From the device a count of 0 and less would divide by the zero that 1 - beta^0 is."""
    with pytest.raises(ValueError, match="step"):
        T.AdamW([torch.zeros(10, device=DEV)], step=-1, capturable=capturable)


# ---- malformed offsets ------------------------------------------------------------------------------


def _back_params(s, go, grad, gw, winners, workspace=None, workspace_bytes=0):
    out = torch.empty(0, device=DEV)
    p = T.BackwardParams()
    p.fwd = capi.make_params(s["table"], s["indices"], s["offsets"], out=out, mode=s["mode"], padding_idx=s["padding_idx"],
                             include_last_offset=s["include_last_offset"])
    p.grad_out, p.grad_out_dtype, p.grad_table_dtype = go.data_ptr(), capi.F32, capi.F32
    p.grad_table = grad.data_ptr()
    p.grad_weights = None if gw is None else gw.data_ptr()
    p.winners = None if winners is None else winners.data_ptr()
    p.workspace = None if workspace is None else workspace.data_ptr()
    p.workspace_bytes = workspace_bytes
    return p


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("mode", [capi.MODE_SUM, capi.MODE_MEAN, capi.MODE_MAX, capi.MODE_SQUARE_SUM])
@pytest.mark.parametrize("n,bags", [(300, 40), (1024, 1), (3000, 300), (20_000, 7), (20_000, 3000)])
def test_malformed_offsets_stay_inside_the_buffers(n, bags, mode, last, idx):
    """Offsets that decrease, or lie before the first lookup or far behind the last, give some gradient: the memory around the
    results and the scratch stays as it was, inputs too, and the next well-formed call gives what it gave before."""
    s, go, _, _ = make_bags(n, 900, 24, [n // bags] * (bags - 1) + [n - n // bags * (bags - 1)], mode=mode, dtype=torch.float32,
                            idx=idx, pad=True, include_last=last)
    go = go.contiguous()
    lib, pad = T._lib(), 4096
    winners = None
    if mode == capi.MODE_MAX:
        winners = T.embedding_bag_winners(s["table"], s["indices"], s["offsets"], padding_idx=s["padding_idx"], include_last_offset=last)
    buf = torch.full((pad + 900 * 24 + pad,), 7.0, device=DEV)
    wbuf = torch.full((pad + n + pad,), 7.0, device=DEV)
    grad, gw = buf[pad:-pad], wbuf[pad:-pad] if mode == capi.MODE_SUM else None
    need = lib.fwd_eb_backward_workspace_size(C.byref(_back_params(s, go, grad, gw, winners)))
    scratch = torch.full((pad + (need + 255) // 256 * 256 + pad,), 5, dtype=torch.uint8, device=DEV)

    def call(offsets):
        t = dict(s, offsets=offsets)
        p = _back_params(t, go, grad, gw, winners, scratch[pad:], need)
        capi.check(lib.fwd_eb_backward(C.byref(p), capi.current_stream_ptr()))
        torch.cuda.synchronize()
        return grad.clone(), None if gw is None else gw.clone()

    good, inputs = call(s["offsets"]), [t.clone() for t in (s["indices"], go, s["table"])]
    far = torch.iinfo(idx)
    g = gen(n + bags)
    anywhere = torch.randint(-2 * n, 3 * n, s["offsets"].shape, generator=g, device=DEV).to(idx)
    extremes = torch.tensor([far.min, far.max, -1, 0, n, n + 1], device=DEV, dtype=idx)[
        torch.randint(0, 6, s["offsets"].shape, generator=g, device=DEV)]
    dented = s["offsets"].clone()
    dented[bags // 2] = 3 * n
    dented[-1] = -5
    for offsets in (s["offsets"].flip(0), anywhere, extremes, dented, torch.full_like(dented, far.max), torch.full_like(dented, far.min)):
        kept = offsets.clone()
        call(offsets)
        for b in (buf, wbuf):
            assert (b[:pad] == 7).all() and (b[-pad:] == 7).all()
        assert (scratch[:pad] == 5).all() and (scratch[-pad:] == 5).all()
        assert torch.equal(offsets, kept) and all(same_bits(a, b) for a, b in zip(inputs, (s["indices"], go, s["table"])))
    again = call(s["offsets"])
    assert same_bits(good[0], again[0]) and (gw is None or same_bits(good[1], again[1]))


# ---- the weights' gradient by itself -----------------------------------------------------------------


@pytest.mark.parametrize("n", [1, 3, 4, 33, 1030, 2370, 9475, 40_003, 80_001])
@pytest.mark.parametrize("dim", [1, 5, 64, 132, 260, 1100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_weights_gradient_by_itself(dtype, dim, n):
    """Numbers of lookups around those that a warp takes at a time; rows of one load a lane and of more; lookups of the padding row,
    outside the table and before the first bag."""
    g = gen(n + dim)
    rows = 500
    table = torch.randn(rows, dim, generator=g, device=DEV).to(dtype)
    idx = torch.randint(-3, rows + 3, (n,), generator=g, device=DEV, dtype=torch.int32)
    off = torch.arange(min(2, n - 1), n, 7, device=DEV, dtype=torch.int32)
    go = torch.randn(off.numel(), dim, generator=g, device=DEV).to(dtype)
    _, gw = T.embedding_bag_backward(go, table, idx, off, padding_idx=7, need_table=False, need_weights=True)
    bag = (torch.arange(n, device=DEV) - off[0]).div(7, rounding_mode="floor")
    keep = (bag >= 0) & (idx >= 0) & (idx < rows) & (idx != 7)
    prod = go.to(F64)[bag.clamp(min=0)] * table.to(F64)[idx.long().clamp(0, rows - 1)] * keep[:, None]
    within(gw, prod.sum(1), (dim + 2) * U * prod.abs().sum(1), "grad_weights")
    assert not gw[~keep].any()


def test_gather_gradient_right_behind_a_compaction():
    """The indices that a window's compaction keeps are read by the next call's first kernel."""
    batches = [make_bags(seed, 900, 64, [40] * 100, mode=capi.MODE_SUM, dtype=torch.float32) for seed in range(6)]
    kept = torch.empty(4000, dtype=torch.int32, device=DEV)
    bounds, pooled = torch.empty(100, 2, dtype=torch.int32, device=DEV), torch.empty(100, 64, device=DEV)
    go = torch.randn(4000, 64, generator=gen(1), device=DEV)

    def run(wait):
        got = []
        for s, _, _, _ in batches * 3:
            window = s["table"][:500]
            kept.fill_(-1)                                   # names no row
            wait()
            capi.compact_window(capi.make_params(window, s["indices"], s["offsets"], out=pooled), kept, bounds)
            wait()
            got.append(T.embedding_bag_backward(go, window, kept, mode=capi.MODE_GATHER)[0])
            wait()
        return got

    want = run(torch.cuda.synchronize)
    got = run(lambda: None)
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, want)) and want[0].any()


@pytest.mark.parametrize("mode", [capi.MODE_MEAN, capi.MODE_MAX])
@pytest.mark.parametrize("bags,rows", [(16, 200), (3000, 20_000)])
def test_a_captured_chain_of_calls_replays(bags, rows, mode):
    """Lookup (with its winners), norm, both gradients and the step, two batches in one graph: three replays leave the bits of
    six steps with a wait after each call."""
    batches = [make_bags(seed, rows, 64, [9] * bags, mode=mode, dtype=torch.float32) for seed in range(2)]

    def made():
        table, w, b = torch.randn(rows, 64, generator=gen(1), device=DEV), torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
        grads = [torch.empty_like(t) for t in (table, w, b)]
        opt = T.AdamW([table, w, b], state_bits=8, capturable=True, **HYPER)
        opt.bind(grads)
        return table, w, b, grads, opt

    def steps(table, w, b, grads, opt, wait):
        for s, go, _, _ in batches:
            winners = None
            if mode == capi.MODE_MAX:
                winners = T.embedding_bag_winners(table, s["indices"], s["offsets"])
                pooled = winners[..., 0].contiguous()
            else:
                pooled = capi.embedding_bag(table, s["indices"], s["offsets"], mode=mode)
            wait()
            y, mean, rstd = T.layer_norm(pooled, w, b, return_stats=True)
            wait()
            gx, gw, gb = T.layer_norm_backward(go, pooled, mean, rstd, w)
            wait()
            T.embedding_bag_backward(gx, table, s["indices"], s["offsets"], mode=mode, winners=winners, grad_table=grads[0])
            wait()
            grads[1].copy_(gw)
            grads[2].copy_(gb)
            opt.step()
            wait()

    eager, captured = made(), made()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(*captured, lambda: None)
    for _ in range(3):
        steps(*eager, torch.cuda.synchronize)
        graph.replay()
    torch.cuda.synchronize()
    assert int(captured[4].step_tensor) == int(eager[4].step_tensor) == 6
    assert all(same_bits(a, b) for a, b in zip(captured[:3], eager[:3]))
    assert all(same_bits(a, b) for a, b in zip(captured[4].exp_avg_sq, eager[4].exp_avg_sq))


# ---- few lookups of a large table ----------------------------------------------------------------


@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 64, 1024])
@pytest.mark.parametrize("mode", [capi.MODE_SUM, capi.MODE_MEAN, capi.MODE_MAX, capi.MODE_SQUARE_SUM, capi.MODE_GATHER])
def test_few_lookups_of_a_large_table(mode, n):
    """Dense gradients of half a gigabyte, whose zeros want the launches of a large call: one run of sorted lookups and more."""
    rows, dim = 4_100_000, 32
    g = gen(n + mode)
    table = torch.zeros(rows, dim, device=DEV)
    named = torch.randint(0, rows, (max(n // 3, 1),), generator=g, device=DEV)
    idx = named[torch.randint(0, named.numel(), (n,), generator=g, device=DEV)]
    table[named] = torch.randn(named.numel(), dim, generator=g, device=DEV)
    lengths = [n // 2, 0, n - n // 2]
    off = torch.tensor([0, n // 2, n // 2], device=DEV, dtype=torch.int32)
    go = torch.randn(n if mode == capi.MODE_GATHER else 3, dim, generator=g, device=DEV)
    winners = T.embedding_bag_winners(table, idx.int(), off) if mode == capi.MODE_MAX and n else None
    if mode == capi.MODE_MAX and not n:
        winners = torch.zeros(3, dim, 2, device=DEV)
    weights = mode == capi.MODE_SUM
    out = torch.full((rows, dim), 7.0, device=DEV)
    _, gw = T.embedding_bag_backward(go, table, idx.int(), None if mode == capi.MODE_GATHER else off, mode=mode, winners=winners,
                                     grad_table=out, need_weights=weights)
    small, to = torch.unique(idx, return_inverse=True)        # the same lookups of a table of the named rows alone
    want, gw_want = T.embedding_bag_backward(go, table[small].contiguous(), to.int(), None if mode == capi.MODE_GATHER else off,
                                             mode=mode, winners=winners, need_weights=weights)
    bag = torch.arange(n, device=DEV) if mode == capi.MODE_GATHER else torch.repeat_interleave(
        torch.arange(3, device=DEV), torch.tensor(lengths, device=DEV))
    # both sums pass at most n additions, each lookup's product as in the formula
    mag = torch.zeros(small.numel(), dim, device=DEV, dtype=F64).index_add_(0, to, go[bag].abs().to(F64))
    if mode == capi.MODE_SQUARE_SUM:
        mag = mag * 2 * table[small].abs().to(F64)
    assert ((out[small].to(F64) - want.to(F64)).abs() <= 2 * (n + 16) * U * mag).all()
    assert int((out != 0).any(1).sum()) == int((want != 0).any(1).sum())
    assert not weights or ((gw - gw_want).abs().to(F64) <= 2 * (dim + 2) * U * (go[bag].abs() * table[idx].abs()).sum(1).to(F64)).all()


# ---- AdamW: states of 8 bits as plain fp32 gives them ---------------------------------------------------


@pytest.mark.parametrize("param,grad,master", [
    (torch.float32, torch.float32, False), (torch.float16, torch.float16, False), (torch.bfloat16, torch.float32, True)])
def test_adamw_states_of_8_bits_are_those_of_plain_fp32(param, grad, master):
    """Three steps over long chunks, short ones, ragged ends and an odd address, against the formulas in torch's elementary
    operations.  One of those more or less fused moves a few codes in a million, by up to an eighth each.  A root or a
    reciprocal is off by an ulp once in 2^18: 110000 blocks have two scales with one of each, and a code follows only
    where its value is next to a border besides."""
    sizes = [9_000_001, 3000, 257, 70_000]
    c = adam_case(11, sizes, param, grad, 8, master, 1)
    c["params"][0], c["grads"][0] = c["params"][0].clone(), c["grads"][0].clone()       # the long one at an even address
    for k in ("m", "v") + (("masters",) if master else ()):
        c[k][0] = c[k][0].clone()
    (b1, b2), least = HYPER["betas"], 2.0 ** -9
    opt = T.AdamW(c["params"], state_bits=8, masters=c["masters"], exp_avg=c["m"], exp_avg_sq=c["v"], exp_avg_scale=c["ms"],
                  exp_avg_sq_scale=c["vs"], **HYPER)
    odd_scales = 0
    for step in range(3):
        held = [[t.clone() for t in c[k]] for k in ("m", "v", "ms", "vs")]
        opt.step(c["grads"], grad_scale=0.7 + step)
        for i, n in enumerate(sizes):
            m8, v8, ms, vs = (h[i] for h in held)
            wide = lambda s: s.repeat_interleave(256)[:n]  # noqa: E731
            g = c["grads"][i].float() * (0.7 + step)
            m = (m8.float() * wide(ms)) * b1 + g * (1 - b1)
            v = (v8.float() * wide(vs)).square() * b2 + (g * g) * (1 - b2)
            for x, code, scale, up in ((m, c["m"][i], c["ms"][i], False), (v.sqrt(), c["v"][i], c["vs"][i], True)):
                pad = torch.zeros(scale.numel() * 256, device=DEV)
                pad[:n] = x
                want = pad.view(-1, 256).abs().amax(1) * (1.0 / 448.0)
                ulps = (want.view(torch.int32) - scale.view(torch.int32)).abs()
                assert int(ulps.max()) <= 1
                odd_scales += int((ulps > 0).sum())
                t = x * wide(torch.where(scale > 0, 1 / scale, torch.zeros_like(scale)))
                t = torch.where(x > 0, t.clamp(min=least), t) if up else t
                assert same_bits(t.clamp(-448, 448).to(torch.float8_e4m3fn), code), (i, step, up)
    assert odd_scales <= 8


@pytest.mark.parametrize("n", [5000, 9_000_001])
def test_adamw_zeros_of_8_bits_are_code_0(n):
    """Elements that never had a gradient: no sign, no smallest code, whichever path their chunk takes; whole blocks of them too."""
    p, g = torch.ones(n, device=DEV), torch.zeros(n, device=DEV)
    g[::600] = 0.5
    g[4::600] = -0.5
    opt = T.AdamW([p], state_bits=8, **dict(HYPER, weight_decay=0.0))
    for _ in range(2):
        opt.step([g])
        for t in (opt.exp_avg[0], opt.exp_avg_sq[0]):
            assert torch.equal(t.view(torch.uint8) != 0, g != 0)
        assert not (opt.exp_avg_sq[0].view(torch.uint8) & 0x80).any()
        assert (p[g == 0] == 1).all() and (p[g != 0] != 1).all()
