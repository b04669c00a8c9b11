"""The training operators on the GPU against plain 64-bit forms.

Tolerances are bounds of the arithmetic, not fitted numbers.  U = 2^-24 is half a step of fp32; a sum of k
fp32 terms is off by at most k * U * (sum of magnitudes) whatever its order; a result is
rounded once to its type, which moves it by at most half a step of that type (`half_step`).
"""
import math
import os

import pytest

torch = pytest.importorskip("torch")

from forward_b200 import capi, training as T  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}   # smallest values
F64 = torch.float64


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def within(got, ref, bound, what):
    """|got - ref| <= bound + one rounding to got's type, elementwise."""
    assert got.shape == ref.shape, what
    g = got.to(F64)
    assert torch.isfinite(g).all(), f"{what}: not finite"
    slack = bound + half_step(got.dtype) * (ref.abs() + bound) + TINY[got.dtype]
    bad = (g - ref).abs() > slack
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by "
                           f"{float(((g - ref).abs() / slack).max()):.3g} times the bound")


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- gradient of the pooled lookup --------------------------------------------------------


def make_bags(seed, rows, dim, lengths, *, mode, dtype, idx=torch.int32, weighted=False, pad=False, hot=0.0, window=0,
              include_last=False, fixed=0):
    g = gen(seed)
    lengths = torch.tensor(lengths, device=DEV, dtype=torch.int64)
    n, bags = int(lengths.sum()), lengths.numel()
    lo = window
    index = torch.randint(lo - (2 if window else 0), lo + rows + (3 if window else 0), (n,), generator=g, device=DEV)
    if hot:
        index = torch.where(torch.rand(n, generator=g, device=DEV) < hot, lo + rows // 2, index)
    padding = -1
    if pad:
        padding = lo + rows // 3
        index = torch.where(torch.rand(n, generator=g, device=DEV) < 0.2, padding, index)
    starts = torch.cumsum(lengths, 0) - lengths
    offsets = torch.cat([starts, starts.new_tensor([n])]) if include_last else starts
    s = dict(table=torch.randn(rows, dim, generator=g, device=DEV).to(dtype), indices=index.to(idx),
             offsets=None if fixed else offsets.to(idx), fixed_len=fixed, mode=mode, padding_idx=padding, row_lo=lo,
             include_last_offset=include_last, per_sample_weights=None)
    if weighted:
        s["per_sample_weights"] = torch.rand(n, generator=g, device=DEV) * 2 - 1
    out_rows = n if mode == capi.MODE_GATHER else bags
    grad_out = torch.randn(out_rows, dim, generator=g, device=DEV).to(dtype)
    bag = torch.arange(n, device=DEV) if mode == capi.MODE_GATHER else torch.repeat_interleave(
        torch.arange(bags, device=DEV), lengths)
    return s, grad_out, bag, starts


def bag_reference(s, grad_out, bag, starts, winners=None, mean_raw=False):
    """(gradient, sum of magnitudes, lookups per row, weights' gradient, its magnitudes), 64 bits, on the CPU."""
    cpu = lambda t: None if t is None else t.cpu()  # noqa: E731
    index, bag, table, go = cpu(s["indices"]).long() - s["row_lo"], cpu(bag), cpu(s["table"]).to(F64), cpu(grad_out).to(F64)
    rows, dim = table.shape
    pad = cpu(s["indices"]).long() == s["padding_idx"] if s["padding_idx"] >= 0 else torch.zeros_like(index, dtype=torch.bool)
    keep = ~pad & (index >= 0) & (index < rows)
    j = torch.arange(index.numel())
    each = go[bag]
    mode = s["mode"]
    if mode == capi.MODE_MEAN:
        counted = torch.ones_like(j) if mean_raw else (~pad).long()
        count = torch.zeros(go.shape[0], dtype=torch.long).index_add_(0, bag, counted)
        each = each / count.clamp(min=1)[bag][:, None]
    elif mode == capi.MODE_MAX:
        pos = cpu(winners).view(torch.int32)[..., 1]
        each = each * (pos[bag] == (j - cpu(starts)[bag])[:, None])
    w = cpu(s["per_sample_weights"])
    gw = gw_mag = None
    if mode == capi.MODE_SUM:
        at = index.clamp(0, max(rows - 1, 0))
        prod = each * (table[at] if rows else torch.zeros_like(each)) * keep[:, None]
        gw, gw_mag = prod.sum(1), prod.abs().sum(1)
    if w is not None:
        each = each * w.to(F64)[:, None]
    ref = torch.zeros(rows, dim, dtype=F64).index_add_(0, index[keep], each[keep])
    mag = torch.zeros(rows, dim, dtype=F64).index_add_(0, index[keep], each[keep].abs())
    if mode == capi.MODE_SQUARE_SUM:
        ref, mag = ref * 2 * table, mag * 2 * table.abs()
    count = torch.zeros(rows, dtype=F64).index_add_(0, index[keep], torch.ones(int(keep.sum()), dtype=F64))
    return ref, mag, count, gw, gw_mag


def check_bag(s, grad_out, bag, starts, *, mean_raw=False, grad_dtype=None, need_weights=None, old=None, grad_table=None):
    winners = None
    if s["mode"] == capi.MODE_MAX:
        winners = T.embedding_bag_winners(s["table"], s["indices"], s["offsets"], fixed_len=s["fixed_len"],
                                          include_last_offset=s["include_last_offset"], padding_idx=s["padding_idx"],
                                          row_lo=s["row_lo"])
    need_weights = s["mode"] == capi.MODE_SUM if need_weights is None else need_weights
    kw = dict(s)
    flags = capi.FLAG_MEAN_RAW_LENGTH if mean_raw else 0
    got, gw = T.embedding_bag_backward(grad_out, kw.pop("table"), kw.pop("indices"), kw.pop("offsets"), **kw, flags=flags,
                                       winners=winners, grad_dtype=grad_dtype, need_weights=need_weights,
                                       grad_table=grad_table, accumulate=old is not None)
    torch.cuda.synchronize()
    ref, mag, count, gw_ref, gw_mag = bag_reference(s, grad_out, bag, starts, winners, mean_raw)
    # a row's sum: as many additions as lookups and at most 12 more where its pieces are joined (padding
    # zeros), two roundings of the coefficient, two of the factor 2 x
    bound = (count[:, None] + 16) * U * mag
    if old is not None:
        bound = bound + U * (old.cpu().to(F64).abs() + mag)
        ref = ref + old.cpu().to(F64)
    within(got.cpu(), ref, bound, "grad_table")
    if need_weights:
        within(gw.cpu(), gw_ref, (s["table"].shape[1] + 2) * U * gw_mag, "grad_weights")
    return got, gw, winners


MODES = [capi.MODE_SUM, capi.MODE_MEAN, capi.MODE_MAX, capi.MODE_SQUARE_SUM, capi.MODE_GATHER]


# calls of one launch, of a sort in one CTA, of a sort by tiles
TIMES = [1, 10, 30]


@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("dim", [1, 3, 8, 40, 64, 128, 200, 256, 520])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("mode", MODES)
def test_bag_gradient(mode, dtype, dim, times):
    lengths = [0, 1, 7, 0, 33, 64, 31, 32, 2, 5, 0] * times
    s, go, bag, starts = make_bags(dim, 37 * times, dim, lengths, mode=mode, dtype=dtype, pad=dim % 2 == 0, hot=0.3)
    check_bag(s, go, bag, starts)


@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("table,grad", [(torch.float32, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("mode", MODES)
def test_bag_gradient_types_apart(mode, table, grad, times):
    """grad_out of another type than the table, the gradient of either's; weights where the mode has them."""
    lengths = [3, 0, 50, 97, 25] * times
    s, go, bag, starts = make_bags(times, 41 * times, 72, lengths, mode=mode, dtype=table, hot=0.2,
                                   weighted=mode == capi.MODE_SUM)
    for out in (table, grad):
        check_bag(s, go.to(grad), bag, starts, grad_dtype=out)


@pytest.mark.parametrize("n,rows,hot", [(1, 1, 0), (31, 1, 0), (32, 1, 0), (33, 2, 0), (64, 1, 0), (1024, 1, 0),
                                        (1056, 1, 0), (3000, 2, 0.9), (70_000, 1, 0), (100_001, 300, 0.6),
                                        (50_000, 70_000, 0.0), (20_000, 17_000_000, 0.1)])
def test_bag_gradient_runs_and_sort_sizes(n, rows, hot):
    """Rows of one lookup, of a run, of thousands of runs; one to four sort passes."""
    dim = 4 if rows > 1_000_000 else 12
    lengths = [n // 3, 0, n - n // 3]
    s, go, bag, starts = make_bags(n, rows, dim, lengths, mode=capi.MODE_SUM, dtype=torch.float32, hot=hot, weighted=True)
    check_bag(s, go, bag, starts)


@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_bag_gradient_windows_and_forms(mode, idx, times):
    """A row window with indices on both sides of it, 64-bit indices, include_last_offset, fixed lengths."""
    lengths = [5] * 40 * times
    for window, last, fixed in ((1000, False, 0), (0, True, 0), (7, False, 5)):
        s, go, bag, starts = make_bags(window, 50, 20, lengths, mode=mode, dtype=torch.float16, idx=idx, pad=True,
                                       window=window, include_last=last and mode != capi.MODE_GATHER, fixed=fixed)
        check_bag(s, go, bag, starts, grad_dtype=torch.float32)


@pytest.mark.parametrize("times", TIMES)
def test_bag_gradient_lookups_outside_every_bag(times):
    """Lookups before the first offset and behind the last (include_last_offset) belong to no bag."""
    g = gen(5)
    n = 100 * times + 1000 * (times > 1)
    table = torch.randn(11, 16, generator=g, device=DEV)
    index = torch.randint(0, 11, (n,), generator=g, device=DEV, dtype=torch.int32)
    edges = [n // 10, n // 10, n // 2, n - 10]
    offsets = torch.tensor(edges, device=DEV, dtype=torch.int32)
    go = torch.randn(3, 16, generator=g, device=DEV)
    w = torch.rand(n, generator=g, device=DEV)
    got, gw = T.embedding_bag_backward(go, table, index, offsets, include_last_offset=True, per_sample_weights=w,
                                       need_weights=True)
    ref, mag = (torch.zeros(11, 16, dtype=F64, device=DEV) for _ in range(2))
    for b in range(3):
        s, e = edges[b], edges[b + 1]
        ref.index_add_(0, index[s:e].long(), w[s:e, None].to(F64) * go[b].to(F64))
        mag.index_add_(0, index[s:e].long(), w[s:e, None].to(F64) * go[b].to(F64).abs())
    within(got, ref, (n + 16) * U * mag, "grad_table")
    assert (gw[:edges[0]] == 0).all() and (gw[edges[3]:] == 0).all() and (gw[edges[0]:edges[3]] != 0).all()


@pytest.mark.parametrize("longest", [700, 2500, 9000])
@pytest.mark.parametrize("mean_raw", [False, True])
def test_bag_gradient_mean_counts(mean_raw, longest):
    lengths = [0, 3, 1, longest, 2, 2]
    s, go, bag, starts = make_bags(3, 9, 24, lengths, mode=capi.MODE_MEAN, dtype=torch.float32, pad=True)
    s["indices"][0:3] = s["padding_idx"]     # a bag of nothing but padding
    check_bag(s, go, bag, starts, mean_raw=mean_raw)


@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("dim", [48, 7, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("mode", [capi.MODE_SUM, capi.MODE_MEAN, capi.MODE_SQUARE_SUM, capi.MODE_MAX])
def test_bag_gradient_accumulates(mode, dtype, dim, times):
    rows = 6000
    s, go, bag, starts = make_bags(8, rows, dim, [90, 0, 77, 1] * times, mode=mode, dtype=dtype, hot=0.3)
    old = torch.randn(rows, dim, generator=gen(9), device=DEV).to(dtype)
    buf = old.clone()
    got, _, _ = check_bag(s, go, bag, starts, old=old, grad_table=buf)
    assert got is buf
    untouched = torch.ones(rows, dtype=torch.bool, device=DEV)
    untouched[s["indices"].long()] = False
    assert untouched.any() and same_bits(buf[untouched], old[untouched])


@pytest.mark.parametrize("times", TIMES)
@pytest.mark.parametrize("offset,stride", [(0, 40), (1, 40), (0, 41), (3, 57), (8, 48)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_bag_gradient_strides(dtype, offset, stride, times):
    """Rows at odd addresses and strides; what lies between and around them stays."""
    def strided(rows, fill):
        flat = torch.full((rows * stride + offset + 64,), fill, dtype=dtype, device=DEV)
        return flat, flat[offset:offset + rows * stride].view(rows, stride)[:, :40]
    rows = 30 if times == 1 else 5000
    s, go, bag, starts = make_bags(offset, rows, 40, [4, 0, 190, 2] * times, mode=capi.MODE_SUM, dtype=dtype)
    _, table = strided(rows, 0.0)
    table.copy_(s["table"])
    _, grad_out = strided(4 * times, 0.0)
    grad_out.copy_(go)
    flat, buf = strided(rows, 7.0)
    s["table"] = table
    check_bag(s, grad_out, bag, starts, grad_table=buf)
    buf.fill_(7.0)
    assert (flat == 7.0).all()


def test_bag_gradient_empty_calls():
    table = torch.randn(5, 8, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    got, gw = T.embedding_bag_backward(torch.randn(3, 8, device=DEV), table, none, off, need_weights=True)
    assert (got == 0).all() and gw.numel() == 0
    old = torch.ones(5, 8, device=DEV)
    T.embedding_bag_backward(torch.randn(3, 8, device=DEV), table, none, off, grad_table=old, accumulate=True)
    assert (old == 1).all()
    got, _ = T.embedding_bag_backward(torch.zeros(0, 8, device=DEV), table, none, none)
    assert (got == 0).all()
    some = torch.tensor([1, 2], dtype=torch.int32, device=DEV)      # lookups, but no bag holds them
    got, gw = T.embedding_bag_backward(torch.zeros(0, 8, device=DEV), table, some, none, need_weights=True)
    assert (got == 0).all() and (gw == 0).all()
    got, gw = T.embedding_bag_backward(torch.randn(1, 8, device=DEV), table[:0], some, off[:1], need_weights=True)
    assert got.shape == (0, 8) and (gw == 0).all()
    _, gw = T.embedding_bag_backward(torch.randn(1, 8, device=DEV), table, some, off[:1], need_table=False, need_weights=True)
    assert gw.shape == (2,)


def test_bag_gradient_padding_row_of_nan_and_infinity():
    """What a skipped lookup would multiply never reaches a result."""
    table = torch.randn(6, 8, device=DEV)
    table[2] = float("nan")
    idx = torch.tensor([0, 2, 5, 2, 9], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    w = torch.tensor([1.0, float("inf"), 2.0, float("nan"), float("nan")], device=DEV)
    go = torch.randn(2, 8, device=DEV)
    got, gw = T.embedding_bag_backward(go, table, idx, off, padding_idx=2, per_sample_weights=w, need_weights=True)
    assert torch.isfinite(got).all() and torch.isfinite(gw).all()
    assert (got[2] == 0).all() and (gw[[1, 3, 4]] == 0).all()
    assert torch.equal(got[0], go[0]) and torch.equal(got[5], 2 * go[0])


def test_bag_gradient_is_deterministic_and_replays():
    """Same bits on every call, on another stream, and from a captured graph on new inputs."""
    s, go, bag, starts = make_bags(1, 500, 128, [40] * 3000, mode=capi.MODE_MEAN, dtype=torch.float16, pad=True, hot=0.3)
    kw = dict(mode=s["mode"], padding_idx=s["padding_idx"])
    buf = torch.empty_like(s["table"])
    call = lambda: T.embedding_bag_backward(go, s["table"], s["indices"], s["offsets"], grad_table=buf, **kw)  # noqa: E731
    first = call()[0].clone()
    for _ in range(3):
        buf.fill_(3.0)
        assert same_bits(call()[0], first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        buf.fill_(3.0)
        assert same_bits(call()[0], first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    other = torch.randn(go.shape, generator=gen(2), device=DEV).half()
    want = T.embedding_bag_backward(other, s["table"], s["indices"], s["offsets"], **kw)[0]
    go.copy_(other)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert same_bits(buf, want)


def test_bag_gradient_against_differences():
    """The pooled sum is linear in the table and in the weights: a difference of two forward calls along a
    direction is the gradient's product with it."""
    s, go, bag, starts = make_bags(4, 30, 24, [3, 8, 0, 15], mode=capi.MODE_SUM, dtype=torch.float32, weighted=True)
    fwd = lambda t, w: (capi.embedding_bag(t, s["indices"], s["offsets"], per_sample_weights=w).to(F64)  # noqa: E731
                        * go.to(F64)).sum()
    got, gw = T.embedding_bag_backward(go, s["table"], s["indices"], s["offsets"],
                                       per_sample_weights=s["per_sample_weights"], need_weights=True)
    d = torch.randn(30, 24, generator=gen(7), device=DEV)
    dw = torch.randn(26, generator=gen(8), device=DEV)
    w = s["per_sample_weights"]
    by_table = (fwd(s["table"] + d, w) - fwd(s["table"] - d, w)) / 2
    by_weight = (fwd(s["table"], w + dw) - fwd(s["table"], w - dw)) / 2
    # every product |go| |w| |x| of the two calls carries at most 16 + 3 roundings
    scale = 24 * 26 * float(go.abs().max()) * 5 * 5
    assert abs(float(by_table - (got.to(F64) * d.to(F64)).sum())) <= 20 * U * scale
    assert abs(float(by_weight - (gw.to(F64) * dw.to(F64)).sum())) <= 20 * U * scale


def test_bag_gradient_winners_of_long_bags():
    """Positions past 255, which are compared whole, next to bags of 255 and 256 lookups and rows without a winner."""
    for dim, dtype in ((24, torch.float16), (5, torch.float32), (64, torch.float32)):
        s, go, bag, starts = make_bags(dim, 900, dim, [255, 256, 257, 1, 0, 4000, 254, 70_000], mode=capi.MODE_MAX, dtype=dtype,
                                       pad=True)
        check_bag(s, go, bag, starts)


def test_bag_gradient_past_32_bits():
    """A table of more than 2^31 elements: rows at both ends of it, zeros everywhere else."""
    rows, dim = 17_000_000, 128
    table = torch.empty(rows, dim, dtype=torch.float16, device=DEV)
    index = torch.tensor([0, rows - 1, rows - 2, rows // 2, rows - 1] * 400, device=DEV)
    go = torch.randn(2000, dim, generator=gen(1), device=DEV).half()
    off = torch.arange(2000, device=DEV)
    got, _ = T.embedding_bag_backward(go, table, index, off)
    want = torch.zeros(5, dim, dtype=F64, device=DEV)
    for k, slot in enumerate((0, 1, 2, 3, 1)):
        want[slot] += go[k::5].to(F64).sum(0)
    for slot, r in enumerate((0, rows - 1, rows - 2, rows // 2)):
        within(got[r], want[slot], 900 * U * 900 * 5, f"row {r}")
        got[r] = 0
    assert not got.view(torch.int16).any()
    acc = torch.zeros_like(got)
    T.embedding_bag_backward(go, table, index, off, grad_table=acc, accumulate=True)
    within(acc[rows - 1], want[1], 900 * U * 900 * 5, "accumulated")


def test_bag_gradient_refusals():
    table, idx = torch.randn(5, 8, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    off, go = torch.zeros(2, dtype=torch.int32, device=DEV), torch.randn(2, 8, device=DEV)
    bad = lambda exc, *a, **k: pytest.raises(exc, T.embedding_bag_backward, *a, **k)  # noqa: E731
    bad(ValueError, go[:1], table, idx, off)
    bad(ValueError, go, table, idx)
    bad(ValueError, go, table, idx, off.long())
    bad(ValueError, go, table, idx, off, accumulate=True)
    bad(ValueError, go, table, idx, off, need_table=False)
    bad(ValueError, go, table, idx, off, grad_table=torch.empty(4, 8, device=DEV))
    bad(ValueError, go, table, idx, off, grad_table=torch.empty(8, 5, device=DEV).t())
    bad(ValueError, go[:, :1].expand(2, 8), table, idx, off)
    bad(TypeError, go.bfloat16(), table, idx, off)
    bad(TypeError, go, table, idx, off, grad_dtype=torch.bfloat16)
    bad(TypeError, go, table, idx.short(), off.short())
    bad(ValueError, go, table, idx, off, per_sample_weights=torch.ones(3, device=DEV))
    bad(capi.FwdEbError, go, table, idx, off, mode=capi.MODE_MAX)
    bad(capi.FwdEbError, go, table, idx, off, mode=capi.MODE_MEAN, need_weights=True)
    bad(ValueError, go, table, idx, off, mode=capi.MODE_MAX, winners=torch.zeros(2, 7, 2, device=DEV))
    bad(ValueError, go, table, idx, off.cpu())


# ---- layer norm ----------------------------------------------------------------------------

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def depth(cols):
    """Additions that a term of a row's sum passes through, at most: in a thread (64, or the loop kernels' share),
    over a warp and over the warps, and the division."""
    return 64 + cols // 1024 + 11


def rows_of(rows, cols, dtype, seed, stride=0, offset=0):
    g = gen(seed)
    wide = cols + stride
    flat = torch.randn(rows * wide + offset, generator=g, device=DEV).to(dtype)
    x = flat[offset:].view(rows, wide)[:, :cols]
    return x


def ln_reference(x, w, b, eps):
    x64 = x.to(F64)
    mean = x64.mean(1, keepdim=True)
    h = x64 - mean
    rstd = (h.square().mean(1, keepdim=True) + eps) ** -0.5
    w64 = torch.ones(x.shape[1], dtype=F64, device=x.device) if w is None else w.to(F64)
    b64 = torch.zeros(x.shape[1], dtype=F64, device=x.device) if b is None else b.to(F64)
    return h * rstd * w64 + b64, mean, rstd, h, w64, b64


def check_ln(x, w, b, eps=1e-5, out=None):
    y, mean, rstd = T.layer_norm(x, w, b, eps=eps, out=out, return_stats=True)
    ref, m, r, h, w64, b64 = ln_reference(x if out is None or out is not x else x, w, b, eps)
    k = depth(x.shape[1])
    x64 = x.to(F64)
    dm = (k + 1) * U * x64.abs().mean(1, keepdim=True)           # the mean's error
    # variance: its own sum, and what a shifted mean adds: mean((h + d)^2) = var + d^2 as sum(h) = 0
    var = h.square().mean(1, keepdim=True)
    dv = (k + 6) * U * (var + dm * dm) + dm * dm + 2 * U * (var + eps)
    rel = 0.5 * dv / (var + eps - dv).clamp(min=1e-300) + 4 * U
    within(mean, m[:, 0], dm[:, 0], "mean")
    within(rstd, r[:, 0], (rel * r)[:, 0], "rstd")
    hw = (h.abs() + dm) * r * w64.abs()
    within(y, ref, r * (1 + rel) * dm * w64.abs() + (rel + 4 * U) * hw + 2 * U * (hw + b64.abs()), "y")
    return y, mean, rstd


def check_ln_backward(gy, x, mean, rstd, w, **kw):
    gx, gw, gb = T.layer_norm_backward(gy, x, mean, rstd, w, **kw)
    rows, cols = x.shape
    x64, g64 = x.to(F64), gy.to(F64)
    r = rstd.to(F64)[:, None]
    h = (x64 - mean.to(F64)[:, None]) * r
    w64 = torch.ones(cols, dtype=F64, device=x.device) if w is None else w.to(F64)
    g = g64 * w64
    a, b = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    if gx is not None:
        k = depth(cols)
        da = (k + 2) * U * g.abs().mean(1, keepdim=True)
        db = (k + 5) * U * (g * h).abs().mean(1, keepdim=True)
        bound = r * (da + h.abs() * db + 8 * U * (g.abs() + a.abs() + (h * b).abs() + h.abs() * db))
        within(gx, r * (g - a - h * b), bound, "grad_x")
    if gw is not None:
        # a column's sum passes at most rows + 64 additions (32 in the last join, the CTA's row groups)
        mag = (g64 * h).abs()
        within(gw, (g64 * h).sum(0), (rows + 64) * U * mag.sum(0) + 4 * U * mag.sum(0), "grad_weight")
        within(gb, g64.sum(0), (rows + 64) * U * g64.abs().sum(0), "grad_bias")
    return gx, gw, gb


LN_COLS = [1, 2, 7, 8, 64, 100, 128, 129, 250, 256, 768, 1000, 1024, 1031, 2000, 4096, 5000, 8192, 12345, 16384, 40000]


@pytest.mark.parametrize("cols", LN_COLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_both_ways(dtype, cols):
    rows = 3 if cols > 5000 else 67
    g = gen(cols)
    x = rows_of(rows, cols, dtype, cols)
    w = torch.randn(cols, generator=g, device=DEV)
    b = torch.randn(cols, generator=g, device=DEV)
    y, mean, rstd = check_ln(x, w, b)
    gy = rows_of(rows, cols, dtype, cols + 1)
    check_ln_backward(gy, x, mean, rstd, w)


@pytest.mark.parametrize("rows", [0, 1, 2, 5, 31, 600, 4099])
@pytest.mark.parametrize("cols", [24, 512, 1500])
def test_layer_norm_row_counts(rows, cols):
    x, gy = rows_of(rows, cols, torch.bfloat16, rows), rows_of(rows, cols, torch.bfloat16, rows + 1)
    w = torch.randn(cols, generator=gen(1), device=DEV).bfloat16()
    y, mean, rstd = check_ln(x, w, None)
    gx, gw, gb = check_ln_backward(gy, x, mean, rstd, w)
    assert gx.shape == (rows, cols) and gw.dtype == torch.bfloat16


@pytest.mark.parametrize("offset,stride", [(0, 0), (1, 0), (0, 3), (5, 7), (8, 8), (4, 4)])
@pytest.mark.parametrize("cols", [48, 1024, 9001, 24000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_layer_norm_strides(dtype, cols, offset, stride):
    rows = 5
    x = rows_of(rows, cols, dtype, 3, stride, offset)
    gy = rows_of(rows, cols, dtype, 4, stride, 0)
    flat = torch.full((rows * (cols + stride) + 64,), 9.0, dtype=dtype, device=DEV)
    out = flat[offset:offset + rows * (cols + stride)].view(rows, cols + stride)[:, :cols]
    w = torch.randn(cols + 1, generator=gen(1), device=DEV)[1:]        # 4 bytes off a 16-byte border
    y, mean, rstd = check_ln(x, w, None, out=out)
    assert y is out
    out.fill_(9.0)
    assert (flat == 9.0).all()
    check_ln_backward(gy, x, mean, rstd, w, grad_x=out)
    out.fill_(9.0)
    assert (flat == 9.0).all()


@pytest.mark.parametrize("wdtype", DTYPES)
def test_layer_norm_weight_forms(wdtype):
    x, gy = rows_of(40, 320, torch.float16, 1), rows_of(40, 320, torch.float16, 2)
    w = torch.randn(320, generator=gen(1), device=DEV).to(wdtype)
    b = torch.randn(320, generator=gen(2), device=DEV).to(wdtype)
    for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
        _, mean, rstd = check_ln(x, ww, bb)
    check_ln_backward(gy, x, mean, rstd, w)
    check_ln_backward(gy, x, mean, rstd, None, param_dtype=wdtype)
    assert check_ln_backward(gy, x, mean, rstd, w, need_params=False)[1:] == (None, None)
    assert check_ln_backward(gy, x, mean, rstd, w, need_x=False)[0] is None


@pytest.mark.parametrize("cols", [64, 3000, 20000])
def test_layer_norm_in_place(cols):
    """y over x; grad_x over grad_y and over x (the column sums must not see it)."""
    x, gy = rows_of(9, cols, torch.float32, 1), rows_of(9, cols, torch.float32, 2)
    w = torch.randn(cols, generator=gen(1), device=DEV)
    y, mean, rstd = T.layer_norm(x, w, return_stats=True)
    gx, gw, gb = T.layer_norm_backward(gy, x, mean, rstd, w)
    a = x.clone()
    assert T.layer_norm(a, w, out=a) is a and same_bits(a, y)
    for over_x in (False, True):
        xx, gg = x.clone(), gy.clone()
        got = T.layer_norm_backward(gg, xx, mean, rstd, w, grad_x=xx if over_x else gg)
        assert all(same_bits(p, q) for p, q in zip(got, (gx, gw, gb)))


def test_layer_norm_far_from_zero_and_constant_rows():
    """A mean a thousand times the spread, a constant row (rstd = eps^-1/2, y = bias), huge and tiny values."""
    x = rows_of(6, 512, torch.float32, 1)
    x[0] += 1000.0
    x[1] = 3.0
    x[2] = 0.0
    x[3] *= 1e15
    x[4] *= 1e-12
    b = torch.randn(512, generator=gen(1), device=DEV)
    y, mean, rstd = check_ln(x, None, b)
    assert torch.equal(y[1], b) and torch.equal(y[2], b)
    assert abs(float(rstd[1]) - 1e-5 ** -0.5) <= 4 * U * 317


def test_layer_norm_nan_stays_in_its_row():
    x = rows_of(8, 200, torch.float32, 1)
    clean = T.layer_norm(x)
    x[3, 5] = float("nan")
    x[6, 0] = float("inf")
    y = T.layer_norm(x)
    rows = [0, 1, 2, 4, 5, 7]
    assert same_bits(y[rows], clean[rows]) and torch.isnan(y[3]).all()


def test_layer_norm_deterministic_and_replays():
    x, gy = rows_of(5000, 256, torch.bfloat16, 1), rows_of(5000, 256, torch.bfloat16, 2)
    w = torch.randn(256, generator=gen(1), device=DEV)
    _, mean, rstd = T.layer_norm(x, w, return_stats=True)
    first = T.layer_norm_backward(gy, x, mean, rstd, w)
    assert all(same_bits(a, b) for a, b in zip(T.layer_norm_backward(gy, x, mean, rstd, w), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean2, rstd2 = T.layer_norm(x, w, return_stats=True)
        got = T.layer_norm_backward(gy, x, mean2, rstd2, w)
    x.copy_(rows_of(5000, 256, torch.bfloat16, 7))
    graph.replay()
    graph.replay()
    y2, m, r = T.layer_norm(x, w, return_stats=True)
    want = T.layer_norm_backward(gy, x, m, r, w)
    assert same_bits(y, y2) and all(same_bits(a, b) for a, b in zip(got, want))


def test_layer_norm_gradient_against_differences():
    """Central differences of the 64-bit formula along random directions."""
    x, gy = rows_of(7, 96, torch.float32, 1), rows_of(7, 96, torch.float32, 2)
    w = torch.randn(96, generator=gen(1), device=DEV)
    b = torch.randn(96, generator=gen(2), device=DEV)
    _, mean, rstd = T.layer_norm(x, w, b, return_stats=True)
    gx, gw, gb = T.layer_norm_backward(gy, x, mean, rstd, w)
    f = lambda x, w, b: (ln_reference(x, w, b, 1e-5)[0] * gy.to(F64)).sum()  # noqa: E731
    e = 1e-5
    x, w, b = x.to(F64), w.to(F64), b.to(F64)
    for which, grad in enumerate((gx, gw, gb)):
        d = torch.randn(grad.shape, generator=gen(which), device=DEV, dtype=F64)
        at = lambda s: f(*[t + (s * d if i == which else 0) for i, t in enumerate((x, w, b))])  # noqa: E731
        diff = float(at(e) - at(-e)) / (2 * e)
        # the difference's own error: e^2 of the third derivative (rstd ~ 1, values of a few), 1e-16 / e of rounding
        assert abs(diff - float((grad.to(F64) * d).sum())) <= 100 * U * float((grad.to(F64) * d).abs().sum()) + 1e-5


def test_layer_norm_past_32_bits():
    x = torch.empty(70_000, 32_768, dtype=torch.bfloat16, device=DEV)
    x[-3:] = rows_of(3, 32_768, torch.bfloat16, 1)
    x[:-3] = 1.0
    y, mean, rstd = T.layer_norm(x, return_stats=True)
    assert same_bits(y[-3:], T.layer_norm(x[-3:].clone())) and not y[:-3].any()
    gy = torch.zeros_like(x)
    gy[-3:] = rows_of(3, 32_768, torch.bfloat16, 2)
    gx, gw, gb = T.layer_norm_backward(gy, x, mean, rstd, grad_x=gy)
    check_ln_backward(rows_of(3, 32_768, torch.bfloat16, 2), x[-3:], mean[-3:], rstd[-3:], None)
    three = rows_of(3, 32_768, torch.bfloat16, 2).to(F64)        # every other row adds zeros
    within(gb, three.sum(0), 3 * U * three.abs().sum(0), "grad_bias")
    assert not gx[:-3].any()


def test_layer_norm_refusals():
    x = torch.randn(4, 16, device=DEV)
    s = torch.ones(4, device=DEV)
    bad = lambda exc, f, *a, **k: pytest.raises(exc, f, *a, **k)  # noqa: E731
    bad(ValueError, T.layer_norm, x[0])
    bad(ValueError, T.layer_norm, x.t())
    bad(ValueError, T.layer_norm, x, torch.ones(15, device=DEV))
    bad(TypeError, T.layer_norm, x, torch.ones(16, device=DEV), torch.ones(16, device=DEV).half())
    bad(TypeError, T.layer_norm, x.double())
    bad(TypeError, T.layer_norm, x, out=x.half())
    bad(ValueError, T.layer_norm, x, out=x[:3])
    bad(ValueError, T.layer_norm, x[:1].expand(4, 16))
    bad(capi.FwdEbError, T.layer_norm, x, eps=-1.0)
    bad(capi.FwdEbError, T.layer_norm, torch.empty(4, 0, device=DEV))
    bad(ValueError, T.layer_norm_backward, x, x, s[:3], s)
    bad(ValueError, T.layer_norm_backward, x, x, s.half(), s)
    bad(TypeError, T.layer_norm_backward, x.half(), x, s, s)
    bad(TypeError, T.layer_norm_backward, x, x, s, s, param_dtype=torch.float64)


# ---- AdamW -----------------------------------------------------------------------------------

HYPER = dict(lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def to_codes(x, up=False):
    """e4m3 codes and scales of the blocks of 256, as the header defines them."""
    n = x.numel()
    pad = torch.zeros(-(-n // 256) * 256, device=DEV)
    pad[:n] = x
    b = pad.view(-1, 256)
    scale = b.abs().amax(1) * (1.0 / 448.0)
    inv = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    t = (b * inv[:, None]).clamp(-448, 448)
    if up:
        t = torch.where(b > 0, t.clamp(min=2.0 ** -9), t)
    return t.view(-1)[:n].to(torch.float8_e4m3fn), scale


def from_codes(code, scale):
    return code.to(F64) * scale.to(F64).repeat_interleave(256)[:code.numel()]


def adam_case(seed, sizes, param, grad, bits, master, offset=0):
    g = gen(seed)
    cut = lambda t: torch.cat([torch.zeros(offset, device=DEV).to(t.dtype), t])[offset:] if offset else t  # noqa: E731
    rnd = lambda n, s: torch.randn(n, generator=g, device=DEV) * s  # noqa: E731
    c = dict(params=[], grads=[], masters=[] if master else None, m=[], v=[], ms=[], vs=[])
    for n in sizes:
        p = rnd(n, 1.0)
        c["params"].append(cut(p.to(param)))
        if master:
            c["masters"].append(cut(p.clone()))
        c["grads"].append(cut(rnd(n, 0.1).to(grad)))
        m, v = rnd(n, 0.05), rnd(n, 0.1).square()
        if bits == 8:
            (m, ms), (v, vs) = to_codes(m), to_codes(v.sqrt(), True)
            c["ms"].append(ms)
            c["vs"].append(vs)
        c["m"].append(cut(m))
        c["v"].append(cut(v))
    return c


def check_adam(c, bits, step, grad_scale, opt_kw=None, step_kw=None, hyper=HYPER):
    lr, (b1, b2), eps, wd = hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"]
    old = {k: [t.clone() for t in v] if v else v for k, v in c.items()}
    opt = T.AdamW(c["params"], state_bits=bits, masters=c["masters"], exp_avg=c["m"], exp_avg_sq=c["v"],
                  exp_avg_scale=c["ms"] or None, exp_avg_sq_scale=c["vs"] or None, step=step - 1, **hyper, **(opt_kw or {}))
    opt.step(c["grads"], **(step_kw or dict(grad_scale=grad_scale)))
    torch.cuda.synchronize()
    for i in range(len(c["params"])):
        g = old["grads"][i].to(F64) * grad_scale
        p = (old["masters"] or old["params"])[i].to(F64)
        if bits == 8:
            m, v = from_codes(old["m"][i], old["ms"][i]), from_codes(old["v"][i], old["vs"][i]).square()
        else:
            m, v = old["m"][i].to(F64), old["v"][i].to(F64)
        m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        # four roundings (two of the constants, two of products) and the sum's; three more where a state is decoded
        dm, dv = 8 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 10 * U * v1
        root = v1.sqrt()
        den = root / math.sqrt(1 - b2 ** step) + eps
        upd = lr / (1 - b1 ** step) * m1 / den
        ref = p * (1 - lr * wd) - upd
        # 16 roundings of the update, the error of m through it, three of the decayed value and the difference
        bound = 16 * U * upd.abs() + lr / (1 - b1 ** step) * dm / den + 4 * U * (p.abs() + upd.abs())
        if c["masters"]:
            within(c["masters"][i], ref, bound, f"master {i}")
            assert same_bits(c["params"][i], c["masters"][i].to(c["params"][i].dtype))
        else:
            within(c["params"][i], ref, bound, f"param {i}")
        if bits == 32:
            within(c["m"][i], m1, dm, f"m {i}")
            within(c["v"][i], v1, dv, f"v {i}")
            continue
        for what, x, code, scale, up in (("m", m1, c["m"][i], c["ms"][i], False), ("v", root, c["v"][i], c["vs"][i], True)):
            n = x.numel()
            pad = torch.zeros(-(-n // 256) * 256, dtype=F64, device=DEV)
            pad[:n] = x.abs()
            top = pad.view(-1, 256).amax(1) / 448
            err = dm if what == "m" else 6 * U * root
            pad[:n] = err
            within(scale, top, pad.view(-1, 256).amax(1) / 448 + 2 * U * top, f"scale of {what} {i}")
            s = scale.to(F64).repeat_interleave(256)[:n]
            got = from_codes(code, scale)
            # half a step of three mantissa bits, half the smallest code (a whole one where zero is avoided)
            slack = 2.0 ** -4 * x.abs() + (2.0 ** -9 if up else 2.0 ** -10) * s + 2 * err + 8 * U * x.abs()
            assert ((got - x).abs() <= slack).all(), f"codes of {what} {i}"
            if up:
                assert (got[(x > 0) & (s > 0)] > 0).all()
    return opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,master", [
    (torch.float32, torch.float32, False), (torch.float16, torch.float16, True), (torch.float16, torch.float32, False),
    (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float16, False), (torch.float32, torch.bfloat16, False)])
def test_adamw_step(bits, param, grad, master):
    sizes = [1, 7, 8, 255, 256, 257, 300, 2048, 4096, 4097, 10_000, 33_333]
    check_adam(adam_case(1, sizes, param, grad, bits, master), bits, step=3, grad_scale=0.25)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 8, 9, 64, 65, 256, 257, 600])
def test_adamw_many_tensors(bits, count):
    sizes = [(i * 37) % 700 for i in range(count)]         # empty ones among them
    check_adam(adam_case(2, sizes, torch.float32, torch.float32, bits, False), bits, step=1, grad_scale=1.0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_adamw_odd_addresses(bits, offset):
    check_adam(adam_case(3, [1000, 5, 4099], torch.float16, torch.float16, bits, True, offset), bits, step=2, grad_scale=2.0)


def test_adamw_leaves_neighbours_alone():
    """Tensors packed side by side in one buffer, a byte or two apart: what lies between stays."""
    flat = {k: torch.full((5000,), 3.0, device=DEV).to(dt) for k, dt in
            (("p", torch.bfloat16), ("g", torch.bfloat16), ("m", torch.float8_e4m3fn), ("v", torch.float8_e4m3fn))}
    spans = [(3, 700), (705, 706), (900, 2900), (2901, 4990)]
    mine = torch.zeros(5000, dtype=torch.bool, device=DEV)
    for a, b in spans:
        mine[a:b] = True
    cut = lambda t: [t[a:b] for a, b in spans]  # noqa: E731
    scales = [[torch.full((-(-(b - a) // 256) + 1,), 5.0, device=DEV) for a, b in spans] for _ in range(2)]
    opt = T.AdamW(cut(flat["p"]), state_bits=8, exp_avg=cut(flat["m"]), exp_avg_sq=cut(flat["v"]),
                  exp_avg_scale=[s[:-1] for s in scales[0]], exp_avg_sq_scale=[s[:-1] for s in scales[1]], **HYPER)
    opt.step(cut(flat["g"]))
    for k in "pmv":
        assert (flat[k].float()[~mine] == 3.0).all()
        assert k != "p" or (flat[k].float()[mine] != 3.0).all()
    assert (flat["g"] == 3.0).all() and all(float(s[-1]) == 5.0 for ss in scales for s in ss)


def test_adamw_zero_states_and_zero_gradients():
    """A first step from nothing; blocks of zeros stay zeros; states far below the normal range do not turn to NaN."""
    p = torch.ones(600, device=DEV)
    g = torch.zeros(600, device=DEV)
    g[300] = 1e-3
    for bits in (32, 8):
        q = p.clone()
        opt = T.AdamW([q], state_bits=bits, **HYPER)
        opt.step([g])
        want = torch.full((600,), 1 - 0.01 * 0.1, device=DEV, dtype=F64)
        want[300] -= 0.01 * 1e-3 / (1e-3 + 1e-8)
        assert ((q.to(F64) - want).abs() <= 32 * U).all()
        assert int((opt.exp_avg[0].float() != 0).sum()) == 1 and int((opt.exp_avg_sq[0].float() != 0).sum()) == 1
    opt.step([torch.full((600,), 1e-37, device=DEV)])
    for _ in range(900):                                    # 0.9^900: through the subnormal range to zero
        opt.step([torch.zeros(600, device=DEV)])
    assert torch.isfinite(q).all() and torch.isfinite(opt.exp_avg[0].float()).all()
    assert torch.isfinite(opt.exp_avg_scale[0]).all() and torch.isfinite(opt.exp_avg_sq_scale[0]).all()


def test_adamw_nonfinite_gradient_stays_in_its_element_or_block():
    for bits in (32, 8):
        p = torch.ones(1024, device=DEV)
        g = torch.full((1024,), 0.5, device=DEV)
        g[300], g[800] = float("nan"), float("inf")
        opt = T.AdamW([p], state_bits=bits, **HYPER)
        opt.step([g])
        bad = ~torch.isfinite(p)
        assert bad[300] and bad[800] and int(bad.sum()) == 2
        opt.step([torch.full((1024,), 0.5, device=DEV)])
        clean = torch.ones(1024, dtype=torch.bool, device=DEV)
        clean[300] = clean[800] = False
        if bits == 8:                       # an infinity takes its block with it, a NaN does not
            clean[768:] = False
        assert torch.isfinite(p[clean]).all() and not torch.isfinite(p[~clean]).any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_device_scalars(bits):
    """step, lr, grad_scale and skip read from the device, and a captured step that counts on with each replay."""
    sizes = [5000, 77]
    c = adam_case(5, sizes, torch.float16, torch.float32, bits, True)
    scale = torch.tensor([0.5], device=DEV)
    check_adam(c, bits, step=7, grad_scale=0.5, opt_kw=dict(capturable=True), step_kw=dict(grad_scale=scale))
    c1, c2 = adam_case(6, sizes, torch.float16, torch.float32, bits, True), adam_case(6, sizes, torch.float16, torch.float32, bits, True)
    mk = lambda c, **kw: T.AdamW(c["params"], state_bits=bits, masters=c["masters"], exp_avg=c["m"], exp_avg_sq=c["v"],  # noqa: E731
                                 exp_avg_scale=c["ms"] or None, exp_avg_sq_scale=c["vs"] or None, step=4, capturable=True, **HYPER)
    skip = torch.zeros(1, dtype=torch.int32, device=DEV)
    a, b = mk(c1), mk(c2)
    b.bind(c2["grads"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step(skip=skip)
    b.step_tensor.fill_(4)                                   # capture ran nothing, but the host counted
    for turn in range(3):
        if turn == 2:
            a.lr_tensor.fill_(0.002)
            b.lr_tensor.fill_(0.002)
        a.step(c1["grads"], skip=skip)
        graph.replay()
    torch.cuda.synchronize()
    assert int(a.step_tensor) == int(b.step_tensor) == 7
    for k in ("params", "masters", "m", "v", "ms", "vs"):
        assert all(same_bits(p, q) for p, q in zip(c1[k], c2[k]))
    before = [t.clone() for t in c2["params"] + c2["m"] + c2["v"]]
    skip.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(same_bits(p, q) for p, q in zip(before, c2["params"] + c2["m"] + c2["v"]))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_32_bits(bits):
    """A tensor of more than 2^31 elements steps at its end as a short one does."""
    n, tail = 2**31 + 5000, 2048 + 136          # the last blocks: the tail starts on a block's border
    assert (n - tail) % 256 == 0
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[-tail:] = torch.randn(tail, generator=gen(1), device=DEV).bfloat16()
    q, h = p[-tail:].clone(), g[-tail:].clone()
    opt, short = (T.AdamW([t], state_bits=bits, **HYPER) for t in (p, q))
    opt.step([g])
    short.step([h])
    assert same_bits(p[-tail:], q) and same_bits(opt.exp_avg_sq[0][-tail:], short.exp_avg_sq[0])
    assert (p[:1000] == p[0]).all() and float(p[0]) == float(torch.tensor(0.5 * (1 - 0.01 * 0.1)).bfloat16())


def test_the_first_call_may_be_captured():
    """Nothing is set up on first use that a stream capture forbids: each operator's first call in a process."""
    import subprocess
    import sys
    code = (
        "import sys, torch; sys.path.insert(0, {root!r})\n"
        "from forward_b200 import training as T\n"
        "x = torch.randn(600, 2000, device='cuda'); w = torch.ones(2000, device='cuda'); s = torch.ones(600, device='cuda')\n"
        "t = torch.randn(5000, 64, device='cuda'); i = torch.zeros(9000, dtype=torch.int32, device='cuda')\n"
        "o = torch.arange(0, 9000, 9, dtype=torch.int32, device='cuda'); go = torch.randn(1000, 64, device='cuda')\n"
        "opt = T.AdamW([t], state_bits=8, capturable=True); opt.bind([torch.ones_like(t)])\n"
        "torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    y = T.layer_norm(x, w); r = T.layer_norm_backward(x, x, s, s, w)\n"
        "    b = T.embedding_bag_backward(go, t, i, o)[0]; c = T.embedding_bag_backward(go[:10], t, i[:90], o[:10])[0]; opt.step()\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert torch.equal(y, T.layer_norm(x, w)) and torch.equal(b, T.embedding_bag_backward(go, t, i, o)[0])\n"
        "assert (b[0] != 0).any() and (c[0] != 0).any()\n"
    ).format(root=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_adamw_refusals():
    p = torch.zeros(10, device=DEV)
    pytest.raises(ValueError, T.AdamW, [p, p])
    m = torch.zeros(10, device=DEV)
    pytest.raises(ValueError, T.AdamW, [p], exp_avg=[m], exp_avg_sq=[m])
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=float("nan"))):
        pytest.raises(capi.FwdEbError, T.AdamW, [p], **kw)
    bad = lambda exc, *a, **k: pytest.raises(exc, T.AdamW, *a, **k)  # noqa: E731
    bad(TypeError, [p.double()])
    bad(ValueError, [torch.zeros(4, 4, device=DEV).t()[1:]])
    bad(ValueError, [p], state_bits=16)
    bad(ValueError, [p], masters=[])
    bad(TypeError, [p.half()], masters=[p.half()])
    bad(ValueError, [p], exp_avg=[torch.zeros(9, device=DEV)])
    bad(TypeError, [p], state_bits=8, exp_avg=[torch.zeros(10, device=DEV)])
    bad(ValueError, [p], exp_avg_scale=[torch.zeros(1, device=DEV)])
    bad(ValueError, [p], weight_decay=[0.1, 0.2])
    opt = T.AdamW([p])
    pytest.raises(ValueError, opt.step)
    pytest.raises(ValueError, opt.step, [p, p])
    pytest.raises(ValueError, opt.step, [p[:9]])
    pytest.raises(ValueError, opt.step, [p.cpu()])
    pytest.raises(TypeError, opt.step, [p.double()])
    g = torch.ones(10, device=DEV)
    pytest.raises(capi.FwdEbError, opt.step, [g], lr=-1.0)
    assert opt.step_count == 0
    opt.step()                                               # the refused lr is not kept
    assert (p < 0).all() and opt.step_count == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pytest.raises(RuntimeError, opt.step)
    pytest.raises(TypeError, opt.step, [p], lr=0.1, skip=torch.zeros(1, device=DEV))
    pytest.raises(TypeError, opt.step, [p], lr=0.1, skip=1)


# ---- together -----------------------------------------------------------------------------------


def test_a_training_step_of_a_table():
    """Lookup -> layer norm -> loss -> the way back -> AdamW on the table and the norm's parameters, three
    steps, against the same in 64 bits with torch's own differentiation."""
    g = gen(11)
    rows, dim, bags = 200, 64, 50
    lengths = torch.randint(0, 9, (bags,), generator=g, device=DEV)
    n = int(lengths.sum())
    off = (torch.cumsum(lengths, 0) - lengths).int()
    idx = torch.randint(0, rows, (n,), generator=g, device=DEV, dtype=torch.int32)
    table = torch.randn(rows, dim, generator=g, device=DEV)
    w, b = torch.ones(dim, device=DEV), torch.zeros(dim, device=DEV)
    target = torch.randn(bags, dim, generator=g, device=DEV)
    leaves = [t.to(F64).requires_grad_() for t in (table, w, b)]
    plain = torch.optim.AdamW(leaves, lr=0.01, betas=(0.9, 0.95), eps=1e-4, weight_decay=0.1)
    grad = torch.empty_like(table)
    gw, gb = torch.empty_like(w), torch.empty_like(b)
    opt = T.AdamW([table, w, b], lr=0.01, betas=(0.9, 0.95), eps=1e-4, weight_decay=0.1)
    opt.bind([grad, gw, gb])
    bag = torch.repeat_interleave(torch.arange(bags, device=DEV), lengths)
    for _ in range(3):
        pooled = capi.embedding_bag(table, idx, off, mode=capi.MODE_MEAN)
        y, mean, rstd = T.layer_norm(pooled, w, b, eps=1e-2, return_stats=True)
        gx, dw, db = T.layer_norm_backward(y - target, pooled, mean, rstd, w)
        T.embedding_bag_backward(gx, table, idx, off, mode=capi.MODE_MEAN, grad_table=grad)
        gw.copy_(dw)
        gb.copy_(db)
        opt.step()

        t64, w64, b64 = leaves
        pool64 = torch.zeros(bags, dim, dtype=F64, device=DEV).index_add_(0, bag, t64[idx.long()])
        pool64 = pool64 / lengths.clamp(min=1)[:, None]
        y64 = torch.nn.functional.layer_norm(pool64, (dim,), w64, b64, 1e-2)
        plain.zero_grad()
        (0.5 * (y64 - target.to(F64)).square().sum()).backward()
        # gradients: a few hundred roundings of values of a few units; after an update with eps = 1e-4 an error of
        # a gradient grows by at most lr / eps = 100 in the parameter, and the next step's gradients carry it
        for got, leaf in ((grad, t64), (gw, w64), (gb, b64)):
            assert float((got.to(F64) - leaf.grad).abs().max()) <= 1e-3 * max(1.0, float(leaf.grad.abs().max()))
        plain.step()
        for got, leaf in zip((table, w, b), leaves):
            assert float((got.to(F64) - leaf.detach()).abs().max()) <= 1e-3


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("n,rows,dim", [(1, 3, 5), (33, 1, 64), (64, 2, 300), (700, 5, 128), (1023, 40, 16), (1024, 1, 8),
                                        (1024, 3000, 1100), (1025, 50, 32), (1025, 1, 8)])
def test_bag_gradient_small_calls(mode, n, rows, dim):
    """Calls that run in one launch, and the first that do not; popular rows, empty bags, many columns."""
    lengths = [n // 2, 0, n - n // 2 - n // 3, 0, n // 3]
    for dtype, weighted in ((torch.float16, False), (torch.float32, mode == capi.MODE_SUM)):
        s, go, bag, starts = make_bags(n + rows, rows, dim, lengths, mode=mode, dtype=dtype, pad=rows > 2, weighted=weighted,
                                       hot=0.4)
        check_bag(s, go, bag, starts)


def test_bag_gradient_small_calls_with_more_bags_than_lookups():
    """Thousands of empty bags around a few lookups, with and without a row that is only padding."""
    lengths = [0] * 3000 + [2, 0, 5] + [0] * 2000 + [1]
    for mode in MODES:
        s, go, bag, starts = make_bags(6, 20, 12, lengths, mode=mode, dtype=torch.float32, pad=True)
        check_bag(s, go, bag, starts)


@pytest.mark.parametrize("param,grad,master", [
    (torch.float16, torch.float16, False), (torch.bfloat16, torch.float32, False), (torch.float32, torch.bfloat16, False),
    (torch.float16, torch.float32, True)])
def test_adamw_8_bits_long_chunks(param, grad, master):
    """Enough elements that a CTA takes several turns with its loads under way; ragged ends, a tensor at an odd address."""
    c = adam_case(4, [9_000_001, 12_345_600, 257], param, grad, 8, master)
    odd = adam_case(5, [4_000_003], param, grad, 8, master, 1)
    for k in c:
        if c[k] is not None:
            c[k] = c[k] + odd[k]
    check_adam(c, 8, step=2, grad_scale=0.5)


def test_adamw_mixed_kinds_in_one_step():
    """Parameters, gradients and master copies of every width side by side, more than one launch covers."""
    cases = [adam_case(7 + i, [300 + 41 * i, 5], p, g, 8, m) for i, (p, g, m) in enumerate(
        (p, g, m) for p in DTYPES for g in DTYPES for m in (False, True) if not (m and p == torch.float32))]
    c = {k: [t for x in cases for t in (x[k] if x[k] is not None else [None] * 2)] for k in cases[0]}
    solo = [T.AdamW(x["params"], state_bits=8, masters=x["masters"], exp_avg=[t.clone() for t in x["m"]],
                    exp_avg_sq=[t.clone() for t in x["v"]], exp_avg_scale=[t.clone() for t in x["ms"]],
                    exp_avg_sq_scale=[t.clone() for t in x["vs"]], **HYPER) for x in
            [{k: [t.clone() if t is not None else None for t in v] if v is not None else None for k, v in x.items()} for x in cases]]
    opt = T.AdamW(c["params"], state_bits=8, masters=c["masters"], exp_avg=c["m"], exp_avg_sq=c["v"], exp_avg_scale=c["ms"],
                  exp_avg_sq_scale=c["vs"], **HYPER)
    opt.step(c["grads"])
    for o, x in zip(solo, cases):
        o.step(x["grads"])
    got = [t for o in solo for t in o.params]
    assert all(same_bits(a, b) for a, b in zip(opt.params, got))
    assert all(same_bits(a, b) for a, b in zip(opt.exp_avg_sq, [t for o in solo for t in o.exp_avg_sq]))


def test_calls_on_two_streams_at_once():
    """Every operator on two streams in turn, nothing waited for in between: the results of one after the other."""
    def work(seed):
        s, go, bag, starts = make_bags(seed, 3000, 64, [30] * 800, mode=capi.MODE_MEAN, dtype=torch.float16, pad=True, hot=0.2)
        small, go2, _, _ = make_bags(seed, 300, 64, [30] * 8, mode=capi.MODE_SUM, dtype=torch.float16)
        x = rows_of(3000, 1000, torch.bfloat16, seed)
        p, g = torch.randn(100_000, generator=gen(seed), device=DEV), torch.randn(100_000, generator=gen(seed + 1), device=DEV)
        opt = T.AdamW([p], state_bits=8, **HYPER)

        def once():
            a = T.embedding_bag_backward(go, s["table"], s["indices"], s["offsets"], mode=s["mode"], padding_idx=s["padding_idx"])[0]
            b = T.embedding_bag_backward(go2, small["table"], small["indices"], small["offsets"])[0]
            y, mean, rstd = T.layer_norm(x, return_stats=True)
            c = T.layer_norm_backward(y, x, mean, rstd)
            opt.step([g])
            return [a, b, y, *c, p.clone()]
        return once

    want = [work(seed)() for seed in (1, 2)]
    calls = [work(1), work(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for k in (0, 1):
        with torch.cuda.stream(streams[k]):
            got[k] = calls[k]()
    again = [[], []]
    for turn in range(6):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                again[k].append(calls[k]())
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(same_bits(a, b) for a, b in zip(got[k], want[k]))
        for r in again[k]:                                   # the parameter moves on, the rest stays
            assert all(same_bits(a, b) for a, b in zip(r[:-1], want[k][:-1]))
