"""What the training operators are measured on: their plain forms, and the calls that take their place.

Three operators that train what the pooled lookup reads:

  bag_grad   the gradient of an EmbeddingBag call: the table's (dense) and the per-sample weights'
  ln_fwd / ln_bwd   layer norm of the pooled rows, and its gradients
  adamw      an AdamW step over many tensors at once, states in 32 or in 8 bits

`own` chooses between the plain torch form and the framework's kernels.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MODES = {"sum": 0, "mean": 1, "max": 2, "square_sum": 3}
NO_POS = 0x7FFFFFFF
BLOCK = 256          # elements that share one scale of an 8-bit state
E4M3_MAX = 448.0
BETAS, EPS, DECAY, LR = (0.9, 0.95), 1e-8, 0.01, 1e-3


# ---- cases ----------------------------------------------------------------------------------

def _bag(name, **kw):
    case = dict(op="bag_grad", rows=1000, dim=64, bags=32, law="uniform", length="fixed", mean_len=20,
                mode="sum", weighted=False, table="f32", accumulate=False, pad=0.0, idx64=False)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _ln(name, op, rows, cols, dtype, affine=True, stride=0, wdtype="f32"):
    case = dict(op=op, rows=rows, cols=cols, dtype=dtype, affine=affine, stride=stride, wdtype=wdtype)
    if name:
        case["name"] = name
    return case


def _adamw(name, tensors, total, param, grad, bits, master, shape_seed=0):
    case = dict(op="adamw", tensors=tensors, total=total, param=param, grad=grad, bits=bits, master=master,
                shape_seed=shape_seed)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one small lookup's gradient (32 bags of 1..20): latency
        _bag("bag_grad_small", rows=10_000, dim=64, bags=32, length="uniform", mean_len=10),
        # the benchmark's lookup: a million rows of 128 halves, 16384 ragged bags, Zipf rows, mean;
        # hot rows gather tens of thousands of lookups, the dense gradient is 256 MB
        _bag("bag_grad_mean_zipf", rows=1_000_000, dim=128, bags=16384, law="zipf", length="poisson",
             mean_len=40, mode="mean", table="f16"),
        # max with padding and empty bags over rows of 512 bytes: one winner a column
        _bag("bag_grad_max_padded", rows=1_000_000, dim=256, bags=8192, length="empty", mean_len=32,
             mode="max", table="f16", pad=0.05),
        # click-model table: 20 weighted lookups a bag, both gradients, added to what is there
        _bag("bag_grad_weighted", rows=4_000_000, dim=128, bags=65536, law="zipf", mean_len=20,
             weighted=True, accumulate=True),
        # the pooled rows of one small request, normalised before its dense layers
        _ln("ln_fwd_small", "ln_fwd", 32, 64, "f32"),
        # the benchmark's pooled rows
        _ln("ln_fwd_pooled", "ln_fwd", 16384, 128, "f16"),
        # a long batch of wide rows, the largest
        _ln("ln_fwd_wide", "ln_fwd", 32768, 4096, "bf16", wdtype="bf16"),
        # the pooled rows on the way back
        _ln("ln_bwd_pooled", "ln_bwd", 16384, 128, "f16"),
        # wide rows on the way back, rows of an odd count and width
        _ln("ln_bwd_wide", "ln_bwd", 16383, 2000, "bf16", wdtype="bf16"),
        # a dense tower's weights and biases: many small tensors, latency
        _adamw("adamw_many_small", 60, 1_500_000, "f32", "f32", 32, False),
        # the benchmark's table with an fp32 master copy, states in 32 bits
        _adamw("adamw_table_32bit", 1, 128_000_000, "f16", "f16", 32, True),
        # 26 tables of ragged sizes, states in 8 bits
        _adamw("adamw_tables_8bit", 26, 100_000_000, "f16", "f16", 8, False, 3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bag_grad", "ln_fwd", "ln_bwd", "adamw"])
    if op == "bag_grad":
        mode = rng.choice(["sum", "sum", "mean", "max", "square_sum"])
        weighted = mode == "sum" and rng.random() < 0.5
        dim = rng.choice([_log_int(rng, 1, 64), 4 * _log_int(rng, 1, 200), 8 * _log_int(rng, 1, 64)])
        rows = min(_log_int(rng, 1, 2_000_000), 128_000_000 // dim)
        mean_len = _log_int(rng, 1, 100)
        most = min(1_000_000, 128_000_000 // dim)
        bags = max(1, min(_log_int(rng, 1, 65536), most // mean_len))
        return _bag(None, rows=rows, dim=dim, bags=bags, law=rng.choice(["uniform", "zipf"]),
                    length=rng.choice(["fixed", "uniform", "poisson", "empty"]), mean_len=mean_len, mode=mode,
                    weighted=weighted, table=rng.choice(["f32", "f16"]), accumulate=rng.random() < 0.3,
                    pad=rng.choice([0.0, 0.05]), idx64=rng.random() < 0.3)
    if op in ("ln_fwd", "ln_bwd"):
        cols = rng.choice([_log_int(rng, 8, 12_000), 8 * _log_int(rng, 1, 1500)])
        rows = max(1, min(_log_int(rng, 1, 100_000), 100_000_000 // cols))
        dtype = rng.choice(["f32", "f16", "bf16"])
        return _ln(None, op, rows, cols, dtype, affine=rng.random() < 0.8,
                   stride=rng.choice([0, 0, 8, 3]), wdtype=rng.choice(["f32", dtype]))
    param = rng.choice(["f32", "f16", "bf16"])
    total = _log_int(rng, 1000, 60_000_000)
    return _adamw(None, min(_log_int(rng, 1, 400), max(1, total // 16)), total, param, rng.choice([param, "f32"]),
                  rng.choice([32, 8]), param != "f32" and rng.random() < 0.5, rng.randrange(1 << 20))


# ---- inputs ---------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _zipf(rows, n, s, g):
    pmf = torch.arange(1, rows + 1, device=DEV, dtype=torch.float64) ** -s
    cdf = torch.cumsum(pmf, 0)
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64) * cdf[-1]
    rank = torch.searchsorted(cdf, u).clamp_(max=rows - 1)
    return torch.randperm(rows, generator=g, device=DEV)[rank]


def _prepare_bag(case, seed):
    g = _gen(seed)
    rows, dim, bags, mean = case["rows"], case["dim"], case["bags"], case["mean_len"]
    if case["length"] == "fixed":
        lengths = torch.full((bags,), mean, device=DEV, dtype=torch.int64)
    else:  # the total is the case's own, whatever the seed, so that the work is too
        low = {"uniform": 1, "poisson": 0, "empty": 0}[case["length"]]
        w = torch.rand(bags, generator=g, device=DEV, dtype=torch.float64)
        if case["length"] == "poisson":
            w = 1 + (w - 0.5) * 2 / math.sqrt(mean)
        free = bags * (mean - low)
        edge = torch.round(torch.cumsum(w, 0) / w.sum().clamp(min=1e-30) * free).long()
        lengths = torch.diff(edge, prepend=edge.new_zeros(1)) + low
    n = bags * mean
    idt = torch.int64 if case["idx64"] else torch.int32
    offsets = torch.cumsum(lengths, 0) - lengths
    index = _zipf(rows, n, 1.05, g) if case["law"] == "zipf" else torch.randint(rows, (n,), generator=g, device=DEV)
    padding = -1
    if case["pad"]:
        padding = 0
        index = torch.where(torch.rand(n, generator=g, device=DEV) < case["pad"], torch.zeros_like(index), index)
    dt = DTYPES[case["table"]]
    s = {"indices": index.to(idt), "padding_idx": padding, "mode": case["mode"], "rows": rows, "dim": dim}
    s["offsets"] = None if case["length"] == "fixed" else offsets.to(idt)
    s["fixed_len"] = mean if case["length"] == "fixed" else 0
    s["grad_out"] = _randn(g, bags, dim).to(dt)
    reads_table = case["weighted"] or case["mode"] == "square_sum"
    table = torch.empty((rows, dim), dtype=dt, device=DEV)
    s["table"] = table.normal_(0, 0.1, generator=g) if reads_table else table
    s["weights"] = torch.rand(n, generator=g, device=DEV) if case["weighted"] else None
    s["winners"] = None
    if case["mode"] == "max":  # {value, position in the bag} a column, as the forward call leaves them
        at = (torch.rand(bags, dim, generator=g, device=DEV) * lengths[:, None]).long()
        none = lengths[:, None] == 0
        if case["pad"]:
            none = none | (index[(offsets[:, None] + at).clamp(max=n - 1)] == padding)
        pair = torch.zeros(bags, dim, 2, device=DEV)
        pair.view(torch.int32)[..., 1] = torch.where(none, torch.full_like(at, NO_POS), at).int()
        s["winners"] = pair
    s["grad_table"] = _randn(g, rows, dim).to(dt) if case["accumulate"] else None
    return s


def _prepare_ln(case, seed):
    g = _gen(seed)
    rows, cols, dt = case["rows"], case["cols"], DTYPES[case["dtype"]]
    wide = cols + case["stride"]
    scale = 0.5 + torch.rand(rows, 1, generator=g, device=DEV)
    s = {"x": (_randn(g, rows, wide) * scale + _randn(g, rows, 1)).to(dt)[:, :cols], "eps": 1e-5,
         "weight": None, "bias": None}
    if case["affine"]:
        wd = DTYPES[case["wdtype"]]
        s["weight"], s["bias"] = (1 + 0.1 * _randn(g, cols)).to(wd), (0.1 * _randn(g, cols)).to(wd)
    if case["op"] == "ln_bwd":
        s["grad_y"] = _randn(g, rows, wide).to(dt)[:, :cols]
        x = s["x"].double()
        s["mean"] = x.mean(1)
        s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + s["eps"]).float()
        s["mean"] = s["mean"].float()
    return s


def _sizes(case):
    """Element counts of the tensors of an adamw case: ragged, their sum near the case's total."""
    r = random.Random(case["shape_seed"])
    share = [math.exp(r.uniform(0, 6)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * x / sum(share))) for x in share]


def _pack(n):
    return -(-n // BLOCK) * BLOCK


def _prepare_adamw(case, seed):
    g = _gen(seed)
    sizes = _sizes(case)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += _pack(n)
    own_part = torch.zeros(at, dtype=torch.bool, device=DEV)
    for a, n in zip(starts, sizes):
        own_part[a:a + n] = True
    flat = lambda scale: torch.where(own_part, _randn(g, at) * scale, 0.0)  # noqa: E731
    s = {"step": 10, "bits": case["bits"], "grad_scale": 0.5}
    full = flat(0.1)
    s["param"] = full.to(DTYPES[case["param"]])
    s["master"] = full if case["master"] else None
    spread = torch.exp2(torch.randint(-6, 1, (at // BLOCK, 1), generator=g, device=DEV).float())
    ragged = lambda t: (t.view(-1, BLOCK) * spread).view(-1)  # noqa: E731
    s["grad"] = ragged(flat(2e-2)).to(DTYPES[case["grad"]])
    m, v = ragged(flat(3e-3)), ragged(flat(1e-2)).square_()
    if case["bits"] == 32:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    else:
        s["m"], s["m_scale"] = _to8(m)
        s["v"], s["v_scale"] = _to8(v.sqrt(), up=True)
    if own:
        from forward_b200 import training

        cut = lambda t: None if t is None else [t[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
        cut_scale = lambda t: None if t is None else [  # noqa: E731
            t[a // BLOCK:a // BLOCK + _pack(n) // BLOCK] for a, n in zip(starts, sizes)]
        s["opt"] = training.AdamW(
            cut(s["param"]), lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
            masters=cut(s["master"]), exp_avg=cut(s["m"]), exp_avg_sq=cut(s["v"]),
            exp_avg_scale=cut_scale(s["m_scale"]), exp_avg_sq_scale=cut_scale(s["v_scale"]), step=s["step"])
        s["opt"].bind(cut(s["grad"]))
    return s


def prepare(case, seed):
    return {"op": case["op"],
            **{"bag_grad": _prepare_bag, "ln_fwd": _prepare_ln, "ln_bwd": _prepare_ln,
               "adamw": _prepare_adamw}[case["op"]](case, seed)}


# ---- plain forms ----------------------------------------------------------------------------

def _to8(x, up=False):
    """e4m3 codes of x with one fp32 scale a block of 256; up: what is above zero stays above zero."""
    b = x.view(-1, BLOCK)
    scale = b.abs().amax(1, keepdim=True) * (1.0 / E4M3_MAX)
    inverse = torch.where(scale > 0, torch.reciprocal(scale), torch.zeros_like(scale))
    t = (b * inverse).clamp(-E4M3_MAX, E4M3_MAX)
    if up:
        t = torch.where(b > 0, t.clamp(min=2.0 ** -9), t)
    return t.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _from8(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _bag_of(s):
    """The bag of every lookup, and every bag's start."""
    n, device = s["indices"].numel(), s["indices"].device
    bags = s["grad_out"].shape[0]
    if s["fixed_len"]:
        start = torch.arange(bags, device=device) * s["fixed_len"]
    else:
        start = s["offsets"].long()
    lengths = torch.diff(start, append=torch.full((1,), n, device=device))
    return torch.repeat_interleave(torch.arange(bags, device=device), lengths, output_size=n), start, lengths


def _plain_bag(s):
    rows, dim = s["rows"], s["dim"]
    dt = s["table"].dtype
    grad = s["grad_out"].float()
    index = s["indices"].long()
    bag, start, lengths = _bag_of(s)
    valid = index != s["padding_idx"]
    into = s["grad_table"] if s["grad_table"] is not None and dt == torch.float32 and s["mode"] != "square_sum" else None
    # few rows take long sums: 64 bits there
    total = into if into is not None else torch.zeros(
        (rows, dim), device=index.device, dtype=torch.float64 if rows * dim <= 1 << 24 else torch.float32)
    grad_w = None
    if s["mode"] == "max":
        pos = s["winners"].view(torch.int32)[..., 1].long()
        has = pos != NO_POS
        at = torch.where(has, start[:, None] + pos, torch.zeros_like(pos))
        cell = index[at] * dim + torch.arange(dim, device=index.device)
        total.view(-1).index_add_(0, cell.view(-1), torch.where(has, grad, torch.zeros_like(grad)).view(-1).to(total.dtype))
    else:
        if s["mode"] == "mean":
            count = torch.zeros(grad.shape[0], device=index.device).index_add_(0, bag, valid.float())
            grad = grad / count.clamp(min=1)[:, None]
        each = grad[bag] * valid[:, None]
        if s["weights"] is not None:
            grad_w = (each * s["table"][index].float()).sum(1)
            each = each * s["weights"][:, None]
        total.index_add_(0, index, each.to(total.dtype))
        if s["mode"] == "square_sum":
            total = total * (2 * s["table"].float())
    if into is not None:
        return [into, grad_w]
    if s["grad_table"] is not None:
        s["grad_table"].copy_(s["grad_table"].float() + total)
        return [s["grad_table"], grad_w]
    return [total.to(dt), grad_w]


def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
    y = centred * rstd
    if s["weight"] is not None:
        y = y * s["weight"].float() + s["bias"].float()
    return [y.to(s["x"].dtype), mean.view(-1), rstd.view(-1)]


def _plain_ln_bwd(s):
    dy = s["grad_y"].float()
    rstd = s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    dw = db = None
    g = dy
    if s["weight"] is not None:
        wt = s["weight"].dtype
        dw, db = (dy * xhat).sum(0).to(wt), dy.sum(0).to(wt)
        g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return [dx.to(s["x"].dtype), dw, db]


def _plain_adamw(s):
    s["step"] += 1
    t, (b1, b2) = s["step"], BETAS
    g = s["grad"].float() * s["grad_scale"]
    m, v = s["m"], s["v"]
    if s["bits"] == 8:
        m, v = _from8(m, s["m_scale"]), _from8(v, s["v_scale"]).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    p = (s["param"] if s["master"] is None else s["master"]).float()
    update = m / (root * (1 / math.sqrt(1 - b2 ** t)) + EPS)
    p = p * (1 - LR * DECAY) - update * (LR / (1 - b1 ** t))
    s["param"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if s["bits"] == 8:
        for name, x, up in (("m", m, False), ("v", root, True)):
            code, scale = _to8(x, up)
            s[name].copy_(code)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return [s["param"], s["master"], s["m"], s["v"], s["m_scale"], s["v_scale"]]


def _own(s):
    from forward_b200 import training

    if s["op"] == "bag_grad":
        return training.embedding_bag_backward(
            s["grad_out"], s["table"], s["indices"], s["offsets"], mode=MODES[s["mode"]], fixed_len=s["fixed_len"],
            per_sample_weights=s["weights"], padding_idx=s["padding_idx"], winners=s["winners"],
            grad_table=s["grad_table"], accumulate=s["grad_table"] is not None,
            need_weights=s["weights"] is not None)
    if s["op"] == "ln_fwd":
        return training.layer_norm(s["x"], s["weight"], s["bias"], eps=s["eps"], return_stats=True)
    if s["op"] == "ln_bwd":
        return training.layer_norm_backward(s["grad_y"], s["x"], s["mean"], s["rstd"], s["weight"],
                                            need_params=s["weight"] is not None)
    s["opt"].step(grad_scale=s["grad_scale"])
    return [s["param"], s["master"], s["m"], s["v"], s["m_scale"], s["v_scale"]]


def run(state):
    if own:
        return list(_own(state))
    return {"bag_grad": _plain_bag, "ln_fwd": _plain_ln_fwd, "ln_bwd": _plain_ln_bwd,
            "adamw": _plain_adamw}[state["op"]](state)


# ---- the definitions, in 64 bits --------------------------------------------------------------

def _exact_bag(s):
    f8 = torch.float64
    n, bags = s["indices"].numel(), s["grad_out"].shape[0]
    index = s["indices"].to(torch.int64)
    j = torch.arange(n, device=index.device)
    begin = j.new_tensor(range(0, n, s["fixed_len"])) if s["fixed_len"] else s["offsets"].to(torch.int64)
    bag = torch.searchsorted(begin, j, right=True) - 1  # the last bag that starts at or before the lookup
    keep = index != s["padding_idx"]
    out = torch.zeros((s["rows"], s["dim"]), dtype=f8, device=index.device)
    dweight = None if s["weights"] is None else torch.zeros(n, dtype=f8, device=index.device)
    count = torch.bincount(bag[keep], minlength=bags).to(f8)
    for a in range(0, n, 1 << 18):
        part = slice(a, min(n, a + (1 << 18)))
        k = keep[part]
        r, b = index[part][k], bag[part][k]
        d = s["grad_out"][b].to(f8)
        if s["mode"] == "mean":
            d = d / count[b][:, None]
        elif s["mode"] == "max":
            d = d * (s["winners"].view(torch.int32)[..., 1][b] == (j[part][k] - begin[b])[:, None])
        elif s["mode"] == "square_sum":
            d = 2 * d * s["table"][r].to(f8)
        if s["weights"] is not None:
            dweight[j[part][k]] = torch.einsum("nd,nd->n", d, s["table"][r].to(f8))
            d = d * s["weights"][part][k].to(f8)[:, None]
        out.index_add_(0, r, d)
    if s["grad_table"] is not None:
        out += s["grad_table"].to(f8)
    return [out, dweight]


def _exact_ln(s, backward):
    f8 = torch.float64
    x = s["x"].to(f8)
    n = x.shape[1]
    w = torch.ones(n, dtype=f8, device=x.device) if s["weight"] is None else s["weight"].to(f8)
    if not backward:
        mu = torch.einsum("rc->r", x) / n
        off = x - mu[:, None]
        r = (torch.einsum("rc,rc->r", off, off) / n + s["eps"]) ** -0.5
        y = torch.einsum("rc,r,c->rc", off, r, w)
        return [y if s["bias"] is None else y + s["bias"].to(f8), mu, r]
    mu, r, dy = s["mean"].to(f8), s["rstd"].to(f8), s["grad_y"].to(f8)
    h = x * r[:, None] - (mu * r)[:, None]
    a = torch.mv(dy, w) / n
    b = torch.einsum("rc,rc,c->r", dy, h, w) / n
    dx = (dy * w - a[:, None] - b[:, None] * h) * r[:, None]
    if s["weight"] is None:
        return [dx, None, None]
    return [dx, torch.einsum("rc,rc->c", dy, h), torch.einsum("rc->c", dy)]


def _exact_adamw(s):
    f8 = torch.float64
    t = s["step"] + 1
    g = s["grad"].to(f8) * s["grad_scale"]
    old_m, old_v = s["m"].to(f8), s["v"].to(f8)
    if s["bits"] == 8:
        old_m = old_m * s["m_scale"].to(f8).repeat_interleave(BLOCK)
        old_v = (old_v * s["v_scale"].to(f8).repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(old_m, g, 1 - BETAS[0])
    v = torch.lerp(old_v, g ** 2, 1 - BETAS[1])
    theta = (s["param"] if s["master"] is None else s["master"]).to(f8)
    theta = theta - LR * DECAY * theta
    theta = theta - LR * (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
    master = None if s["master"] is None else theta
    if s["bits"] == 8:  # the codes round what has 32 bits: the scales have a value in 64, they have none
        peak = lambda z: torch.amax(torch.abs(z).view(-1, BLOCK), 1) / E4M3_MAX  # noqa: E731
        return [theta, master, None, None, peak(m), peak(torch.sqrt(v))]
    return [theta, master, m, v, None, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "bag_grad":
        return _exact_bag(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    return _exact_ln(s, case["op"] == "ln_bwd")


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    if case["op"] == "bag_grad":
        n, e, dim = case["bags"] * case["mean_len"], SIZE[case["table"]], case["dim"]
        ints = (8 if case["idx64"] else 4) * (n + (0 if case["length"] == "fixed" else case["bags"]))
        size = ints + case["bags"] * dim * e
        touched = min(case["rows"], n)
        if case["accumulate"]:  # rows that no lookup names stay as they are; at most one row a lookup
            if case["law"] == "zipf":  # expected distinct rows of the draw
                h = [k ** -1.05 for k in range(1, min(case["rows"], 200_000) + 1)]
                tail = (200_000 ** -0.05 - case["rows"] ** -0.05) / 0.05 if case["rows"] > 200_000 else 0.0
                z = sum(h) + tail
                touched = sum(-math.expm1(-n * x / z) for x in h) + n * tail / z
            else:
                touched = -case["rows"] * math.expm1(-n / case["rows"])
            size += 2 * touched * dim * e
        else:
            size += case["rows"] * dim * e
        if case["weighted"]:
            size += 8 * n + min(touched, n) * dim * e
        if case["mode"] == "max":
            size += case["bags"] * dim * 8
        if case["mode"] == "square_sum":
            size += min(touched, n) * dim * e
        return {"bytes": size, "flops": (4 if case["weighted"] else 2) * n * dim}
    if case["op"] in ("ln_fwd", "ln_bwd"):
        cells, e = case["rows"] * case["cols"], SIZE[case["dtype"]]
        par = case["cols"] * SIZE[case["wdtype"]] * (case["affine"] and 1)
        if case["op"] == "ln_fwd":
            return {"bytes": 2 * cells * e + 2 * par + 8 * case["rows"], "flops": 8 * cells}
        return {"bytes": 3 * cells * e + 3 * par + 8 * case["rows"], "flops": 14 * cells}
    n = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    weight = SIZE[case["param"]] + 8 if case["master"] else 2 * SIZE[case["param"]]
    return {"bytes": n * (state + weight + SIZE[case["grad"]]), "flops": 16 * n}
