"""The row operators of the package -- `layer_norm`, `label_loss`, `sample_labels` -- as cases to be timed and checked.

Every operator works on rows [B, T, C]: a batch of B utterances (or sequences) of T frames (or one token) with C classes (or
channels), `lengths` [B] of which hold something.  `run` computes a case in plain torch (`own = False`) or by the package's
entry points (`own = True`); `exact` is the definition in 64 bits."""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- cases -----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one step of 16 live streams: a row of embeddings each, where only the call's latency counts
        dict(name="norm_step", op="norm", train=False, B=16, T=1, C=512, dtype="bfloat16", wtype="bfloat16", pitch=0, ragged=False),
        # one padded chunk of 16 segments of up to 30 s (the aligner's call shape), embeddings of 768 channels, full precision
        dict(name="norm_chunk", op="norm", train=True, B=16, T=1870, C=768, dtype="float32", wtype="float32", pitch=0, ragged=True),
        # an odd width in rows of a wider buffer: every row starts at another alignment
        dict(name="norm_odd", op="norm", train=True, B=24, T=500, C=1001, dtype="float16", wtype="float32", pitch=1007, ragged=True),
        # a training step of a large model
        dict(name="norm_wide", op="norm", train=True, B=32, T=1024, C=4096, dtype="bfloat16", wtype="bfloat16", pitch=0, ragged=False),
        # one chunk of 16 segments, phoneme head, through autograd
        dict(name="loss_chunk", op="loss", form="autograd", B=16, T=1870, C=67, dtype="float32", pitch=0, ragged=True, weighted=False),
        # a word-piece head of odd width on a few utterances, every row's loss
        dict(name="loss_odd", op="loss", form="none", B=7, T=911, C=5003, dtype="float16", pitch=0, ragged=True, weighted=False),
        # the headline batch, frames weighted by their confidence, loss and gradient of the phoneme head in one go
        dict(name="loss_frames", op="loss", form="fused", B=4096, T=1000, C=67, dtype="float32", pitch=0, ragged=False, weighted=True),
        # a language model's vocabulary
        dict(name="loss_vocab", op="loss", form="fused", B=8, T=1024, C=131072, dtype="bfloat16", pitch=0, ragged=False, weighted=False),
        # one step of eight sequences with parameters of their own
        dict(name="sample_step", op="sample", B=8, T=1, C=32000, dtype="float32", pitch=0, ragged=False, params="each", peak=4.0,
             masked=0.0),
        # one step of a large serving batch, some classes forbidden
        dict(name="sample_vocab", op="sample", B=512, T=1, C=131072, dtype="bfloat16", pitch=0, ragged=False, params="each", peak=4.0,
             masked=0.01),
        # the group head of a padded batch
        dict(name="sample_groups", op="sample", B=300, T=1500, C=17, dtype="float16", pitch=0, ragged=True, params="top_k", peak=3.0,
             masked=0.0),
        # the phoneme head of the headline batch, rows padded to 68 floats as window stitching leaves them
        dict(name="sample_frames", op="sample", B=4096, T=1000, C=67, dtype="float32", pitch=68, ragged=False, params="top_p", peak=6.0,
             masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "loss", "sample"))
    dtype = rng.choice(tuple(_TYPES))
    narrow = rng.random() < 0.5
    if op == "norm":
        C, cap = _log_int(rng, 17, 16384), 1 << 27
    elif narrow:
        C, cap = rng.choice((17, 67, _log_int(rng, 2, 1024))), 1 << 28
    else:
        C, cap = _log_int(rng, 1025, 160000), 1 << (29 if op == "loss" else 26)
    rows = _log_int(rng, 1, max(1, min(4096000, cap // C)))
    B = _log_int(rng, 1, min(rows, 4096))
    T = max(1, rows // B)
    case = dict(op=op, B=B, T=T, C=C, dtype=dtype, pitch=rng.choice((0, 0, C + rng.randint(1, 9))), ragged=rng.random() < 0.5)
    if op == "norm":
        case.update(train=rng.random() < 0.75, wtype=rng.choice((dtype, "float32")))
    elif op == "loss":
        case.update(form=rng.choice(("fused", "autograd", "none")), weighted=rng.random() < 0.5)
    else:
        case.update(params=rng.choice(("each", "plain", "top_k", "top_p", "min_p")), peak=rng.choice((3.0, 4.0, 6.0, 9.0)),
                    masked=rng.choice((0.0, 0.01, 0.3)))
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _rows(case, g, scale=1.0, pitch=None):
    """[B, T, C] normal numbers of the case's type, a view into rows of `pitch` elements where the case has one"""
    pitch = max(case["pitch"], case["C"]) if pitch is None else pitch
    store = torch.empty((case["B"], case["T"], pitch), dtype=_TYPES[case["dtype"]], device="cuda")
    store.normal_(0.0, scale, generator=g)
    return store[..., :case["C"]]


def _spoken(case, x, labels, peak):
    """what a head answers with: `peak` on top of the frame's own class"""
    return x.scatter_add_(2, labels.long().unsqueeze(2), torch.full((1, 1, 1), peak, dtype=x.dtype, device="cuda").expand(
        case["B"], case["T"], 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, C = case["B"], case["T"], case["C"]
    state = dict(case=case, lengths=None)
    if case["ragged"]:
        lengths = torch.randint(max(1, T // 10), T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = T
        state["lengths"] = lengths
    if case["op"] == "norm":
        wt = _TYPES[case["wtype"]]
        state["x"] = _rows(case, g, 1.5).add_(0.25)
        state["weight"] = torch.empty(C, dtype=wt, device="cuda").normal_(1.0, 0.1, generator=g)
        state["bias"] = torch.empty(C, dtype=wt, device="cuda").normal_(0.0, 0.1, generator=g)
        if case["train"]:
            state["grad"] = _rows(case, g, 1.0, C)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_()
    elif case["op"] == "loss":
        state["labels"] = torch.randint(0, C, (B, T), generator=g, device="cuda", dtype=torch.int32)
        state["logits"] = _spoken(case, _rows(case, g), state["labels"], 6.0)
        # some frames are blank to the aligner: it gives them no label
        state["labels"].masked_fill_(torch.rand((B, T), generator=g, device="cuda") < 0.05, -1)
        state["weights"] = torch.rand((B, T), generator=g, device="cuda") if case["weighted"] else None
        if case["form"] == "autograd":
            state["logits"].requires_grad_()
    else:
        labels = torch.randint(0, C, (B, T), generator=g, device="cuda", dtype=torch.int32)
        x = _spoken(case, _rows(case, g, 1.0 if C <= 1024 else 2.0), labels, case["peak"])
        if case["masked"]:
            x.masked_fill_((torch.rand((1, 1, C), generator=g, device="cuda") < case["masked"]), -math.inf)
        state["logits"] = x
        state["uniform"] = torch.rand((B, T), generator=g, device="cuda")
        state["params"] = dict(plain={}, top_k=dict(temperature=0.9, top_k=5), top_p=dict(temperature=0.8, top_p=0.95),
                               min_p=dict(temperature=1.3, min_p=0.05), each=None)[case["params"]]
        if state["params"] is None:  # every sequence brings its own
            pick = lambda values, dt: torch.tensor(values, dtype=dt, device="cuda")[  # noqa: E731
                torch.randint(0, len(values), (B,), generator=g, device="cuda")]
            state["params"] = dict(temperature=pick((0.0, 0.6, 0.8, 1.0, 1.2), torch.float32), top_k=pick((0, 1, 20, 50), torch.int32),
                                   top_p=pick((0.5, 0.9, 0.95, 1.0), torch.float32), min_p=pick((0.0, 0.0, 0.02, 0.1), torch.float32))
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------

EPS = 1e-5


def run(state):
    case = state["case"]
    if own:
        import bournemouth_forced_aligner_amd as bfa
        if case["op"] == "norm":
            y = bfa.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, lengths=state["lengths"])
            if not case["train"]:
                return y
            return [y.detach(), *torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["grad"])]
        if case["op"] == "loss":
            args = dict(weights=state["weights"], lengths=state["lengths"])
            if case["form"] == "fused":
                return list(bfa.label_loss_and_grad(state["logits"], state["labels"], **args))
            if case["form"] == "none":
                return bfa.label_loss(state["logits"], state["labels"], reduction="none", **args)
            loss = bfa.label_loss(state["logits"], state["labels"], **args)
            return [loss.detach(), *torch.autograd.grad(loss, (state["logits"],))]
        return list(bfa.sample_labels(state["logits"], state["uniform"], lengths=state["lengths"], **state["params"]))
    with torch.no_grad():
        return {"norm": _plain_norm, "loss": _plain_loss, "sample": _plain_sample}[case["op"]](state)


def _held(state):
    """[B, T] which rows hold something"""
    B, T = state["case"]["B"], state["case"]["T"]
    if state["lengths"] is None:
        return torch.ones((B, T), dtype=torch.bool, device="cuda")
    return torch.arange(T, device="cuda")[None, :] < state["lengths"][:, None]


def _plain_norm(state):
    held = _held(state)[..., None]
    x, w, b = state["x"], state["weight"].float(), state["bias"].float()
    xf = torch.where(held, x.float(), 0.0)
    d = xf - xf.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    xh = d * r
    y = torch.where(held, xh * w + b, 0.0).to(x.dtype)
    if not state["case"]["train"]:
        return y
    dy = torch.where(held, state["grad"].float(), 0.0)
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    C = x.shape[-1]
    return [y, dx.to(x.dtype), (dy * xh).reshape(-1, C).sum(0).to(state["weight"].dtype),
            dy.reshape(-1, C).sum(0).to(state["bias"].dtype)]


def _plain_loss(state):
    case, z, labels = state["case"], state["logits"], state["labels"].long()
    counts = _held(state) & (labels >= 0)
    zf = z.float()
    e = torch.exp(zf - zf.amax(-1, keepdim=True))
    s = e.sum(-1, keepdim=True)
    at = labels.clamp(min=0)[..., None]
    nll = (zf.amax(-1, keepdim=True) + torch.log(s) - zf.gather(2, at))[..., 0]
    w = torch.where(counts, 1.0 if state["weights"] is None else state["weights"], 0.0)
    nll = torch.where(counts, w * nll, 0.0)
    if case["form"] == "none":
        return nll
    total = w.double().sum()
    inv = torch.where(total > 0, 1.0 / total, 0.0)
    loss = (nll.double().sum() * inv).float()
    scale = (w.double() * inv).float()[..., None]
    e = e / s
    e.scatter_add_(2, at, torch.full((1, 1, 1), -1.0, device="cuda").expand(at.shape))
    return [loss, torch.where(counts[..., None], e * scale, 0.0).to(z.dtype)]


def _per_row(value, case, dtype):
    """a parameter as [B * T, 1] in 64 bits, rounded to the type that the call takes"""
    t = torch.as_tensor(value, device="cuda").to(dtype)
    t = t.expand(case["B"]) if t.dim() == 0 else t
    return t[:, None].expand(case["B"], case["T"]).reshape(-1, 1).to(torch.float64 if dtype.is_floating_point else torch.int64)


def _plain_sample(state):
    """in 64 bits: which class a number falls to is decided at the borders between them"""
    case, z = state["case"], state["logits"]
    C, rows = case["C"], case["B"] * case["T"]
    z, u, held = z.reshape(rows, C), state["uniform"].reshape(rows, 1).double(), _held(state).reshape(rows)
    p = state["params"]
    temp = _per_row(p.get("temperature", 1.0), case, torch.float32)
    top_k = _per_row(p.get("top_k", 0), case, torch.int32)
    top_p = _per_row(p.get("top_p", 1.0), case, torch.float32)
    min_p = _per_row(p.get("min_p", 0.0), case, torch.float32)
    labels = torch.empty(rows, dtype=torch.int32, device="cuda")
    logp = torch.empty(rows, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // C)
    place = torch.arange(C, device="cuda")[None, :]
    for i in range(0, rows, step):
        s = slice(i, min(rows, i + step))
        v = z[s].double()
        v = torch.where(torch.isnan(v), -math.inf, v)
        v, order = torch.sort(v, dim=1, descending=True, stable=True)
        top = v[:, :1]
        t = temp[s]
        x = torch.where(v == top, 0.0, torch.where(t > 0, (v - top) / t, -math.inf))
        w = torch.exp(x)
        keep = (place < top_k[s]) | (top_k[s] <= 0)
        run_sum = torch.cumsum(w * keep, 1)
        keep &= ((run_sum - w * keep) < top_p[s] * run_sum[:, -1:]) | (top_p[s] >= 1)
        keep &= w >= min_p[s]
        keep &= (place == 0) | (t > 0)
        keep[:, 0] = True
        w = w * keep
        in_order = torch.empty_like(w).scatter_(1, order, w)
        mass = torch.cumsum(in_order, 1)
        # the first class whose mass passes the target
        at = (mass <= u[s] * mass[:, -1:]).sum(1, keepdim=True).clamp(max=C - 1)
        xi = torch.empty_like(x).scatter_(1, order, x).gather(1, at)[:, 0]
        none = torch.isneginf(top[:, 0]) | ~held[s]
        labels[s] = torch.where(none, -1, at[:, 0]).int()
        logp[s] = torch.where(none, 0.0, xi - torch.log(mass[:, -1])).float()
    return [labels.view(case["B"], case["T"]), logp.view(case["B"], case["T"])]


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------

def work(case):
    B, T, C = case["B"], case["T"], case["C"]
    out = B * T * C
    n = int(out * (0.55 if case["ragged"] else 1.0))  # lengths are spread evenly over T / 10 ... T; rows behind them are not read
    size = torch.empty((), dtype=_TYPES[case["dtype"]]).element_size()
    if case["op"] == "norm":
        w = torch.empty((), dtype=_TYPES[case["wtype"]]).element_size() * C
        if case["train"]:  # x, dy, w, b -> y, dx, dw, db
            return dict(bytes=2 * (n + out) * size + 4 * w, flops=22 * n)
        return dict(bytes=(n + out) * size + 2 * w, flops=8 * n)
    if case["op"] == "loss":  # logits, labels, weights -> every row's loss, or the gradient
        given = n * size + B * T * (8 if case["weighted"] else 4)
        if case["form"] == "none":
            return dict(bytes=given + B * T * 4, flops=5 * n)
        return dict(bytes=given + out * size, flops=8 * n)
    return dict(bytes=n * size + B * T * 12, flops=8 * n)  # logits, numbers -> labels, their logarithms


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        if case["op"] == "norm":
            return _exact_norm(case, state)
        if case["op"] == "loss":
            return _exact_loss(case, state)
        return _exact_sample(case, state)


def _blocks(case, budget=1 << 26):
    """utterances in ranges of at most about `budget` elements, each cut to ranges of frames where one alone is longer"""
    nb = max(1, budget // (case["T"] * case["C"]))
    nt = case["T"] if case["T"] * case["C"] <= budget else max(1, budget // case["C"])
    for b in range(0, case["B"], nb):
        for t in range(0, case["T"], nt):
            yield slice(b, min(b + nb, case["B"])), slice(t, min(t + nt, case["T"]))


def _frames(case, state, b, t):
    """which of the rows in the block count"""
    last = torch.full((case["B"],), case["T"], device="cuda") if state["lengths"] is None else state["lengths"].long()
    return torch.arange(case["T"], device="cuda")[t].unsqueeze(0) < last[b].unsqueeze(1)


def _exact_norm(case, state):
    B, T, C = case["B"], case["T"], case["C"]
    w, b0 = state["weight"].double(), state["bias"].double()
    y = torch.zeros((B, T, C), dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(y) if case["train"] else None
    dw, db = torch.zeros_like(w), torch.zeros_like(b0)
    for b, t in _blocks(case):
        m = _frames(case, state, b, t)
        rows = state["x"][b, t][m].double()
        var, mu = torch.var_mean(rows, dim=1, correction=0, keepdim=True)
        hat = (rows - mu) * (var + EPS).rsqrt()
        y[b, t][m] = torch.addcmul(b0, hat, w)
        if case["train"]:
            gy = state["grad"][b, t][m].double()
            dw += torch.einsum("rc,rc->c", gy, hat)
            db += gy.sum(0)
            gh = gy * w
            # d(hat)/dx is rstd times the projection that takes out the mean and the part along hat
            gx = gh - gh.mean(1, keepdim=True)
            gx = gx - hat * ((hat * gh).sum(1, keepdim=True) / C)
            dx[b, t][m] = gx * (var + EPS).rsqrt()
    return [y, dx, dw, db] if case["train"] else y


def _exact_loss(case, state):
    B, T, C = case["B"], case["T"], case["C"]
    labels = state["labels"].long()
    weights = torch.ones((B, T), dtype=torch.float64, device="cuda") if state["weights"] is None else state["weights"].double()
    each = torch.zeros((B, T), dtype=torch.float64, device="cuda")
    grad = None if case["form"] == "none" else torch.zeros((B, T, C), dtype=torch.float64, device="cuda")
    denominator = torch.zeros((), dtype=torch.float64, device="cuda")
    for b, t in _blocks(case):
        denominator += weights[b, t][_frames(case, state, b, t) & (labels[b, t] >= 0)].sum()
    for b, t in _blocks(case):
        m = _frames(case, state, b, t) & (labels[b, t] >= 0)
        rows, at, wt = state["logits"][b, t][m].double(), labels[b, t][m], weights[b, t][m]
        lp = torch.log_softmax(rows, dim=1)
        each[b, t][m] = -lp[torch.arange(at.numel(), device="cuda"), at] * wt
        if grad is not None:
            gz = lp.exp()
            gz[torch.arange(at.numel(), device="cuda"), at] -= 1.0
            grad[b, t][m] = gz * (wt / denominator).unsqueeze(1)
    if grad is None:
        return each
    return [each.sum() / denominator if float(denominator) > 0 else torch.zeros_like(denominator), grad]


def _exact_sample(case, state):
    """class i is kept when the classes in front of it (a greater value, or the same and a lower index) are fewer than top_k, hold
    less than top_p of the first top_k's mass, and its own weight reaches min_p"""
    B, T, C = case["B"], case["T"], case["C"]
    if C > 1024 and B * T * C > 1 << 27:
        return None
    prm = {k: torch.as_tensor(state["params"].get(k, v), device="cuda") for k, v in
           dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0).items()}
    prm = {k: (v.to(torch.int32).long() if k == "top_k" else v.to(torch.float32).double()).expand(B) for k, v in prm.items()}
    labels = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    logp = torch.zeros((B, T), dtype=torch.float64, device="cuda")
    for b, t in _blocks(case, 1 << 24):
        m = _frames(case, state, b, t)
        z = state["logits"][b, t][m].double()
        if z.shape[0] == 0:
            continue
        z = torch.nan_to_num(z, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        u = state["uniform"][b, t][m].double()
        temp, k, p, q = (prm[n][b].unsqueeze(1).expand(m.shape)[m] for n in ("temperature", "top_k", "top_p", "min_p"))
        best = z.max(1).values
        dist = torch.where(z < best[:, None], best[:, None] - z, torch.zeros_like(z))
        w = torch.exp(-dist / temp.clamp(min=1e-300)[:, None])
        k = torch.where(k <= 0, torch.full_like(k, C), k)
        if C <= 128:
            # every pair of classes, a few rows at a time
            front_n, front_m = torch.empty_like(z), torch.empty_like(z)
            lower = torch.arange(C, device="cuda")[:, None] < torch.arange(C, device="cuda")[None, :]
            top_mass = torch.empty_like(best)
            step = max(1, (1 << 27) // (C * C))
            for i in range(0, z.shape[0], step):
                r = slice(i, i + step)
                zi, zj = z[r, :, None], z[r, None, :]
                ahead = ((zi > zj) | ((zi == zj) & lower)).double()  # [rows, i, j]: i stands in front of j
                front_n[r] = ahead.sum(1)
                front_m[r] = (ahead * w[r, :, None]).sum(1)
                top_mass[r] = torch.where(front_n[r] < k[r, None], w[r], 0.0).sum(1)
        else:
            front_n, front_m = torch.empty_like(z), torch.empty_like(z)
            order = torch.argsort(-z, dim=1, stable=True)
            ws = w.gather(1, order)
            front_n.scatter_(1, order, torch.arange(C, device="cuda", dtype=torch.float64).expand(z.shape))
            front_m.scatter_(1, order, ws.cumsum(1) - ws)
            top_mass = torch.where(front_n < k[:, None], w, 0.0).sum(1)
        kept = (front_n < k[:, None]) & ((front_m < (p * top_mass)[:, None]) | (p >= 1)[:, None]) & (w >= q[:, None])
        kept = (kept & (temp > 0)[:, None]) | (front_n == 0)
        mass = torch.where(kept, w, 0.0)
        total = mass.sum(1)
        at = (mass.cumsum(1) > (u * total)[:, None]).int().argmax(1)
        none = torch.isneginf(best)
        labels[b, t][m] = torch.where(none, -1, at).int()
        logp[b, t][m] = torch.where(none, 0.0, w.gather(1, at[:, None])[:, 0].log() - total.log())
    return [labels, logp]
