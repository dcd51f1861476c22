"""Cases of the operators around a network's output, for timing them and holding them to their definitions.

Four operators, on matrices of one row per frame (or per token):

  ln       layer norm of every row and its derivatives, those of the scale and the offset (sums over all rows) included
  affine   an affine layer in half precision with its activation and the residual that is added to it, and its derivatives
           with respect to the input, the weights and the bias
  labels   the log-probability of one given label per row, with the row's entropy and its best alternatives; and the
           derivative of the first two with respect to the matrix
  distill  the distillation objective: a row's log-softmax at a temperature against a teacher's top logits, a few (value,
           column) pairs per row; alone (a validation pass) or with its derivative (a training pass)

`run` computes them with elementary torch operations in 32 bits, or with the package's operators where `own` is true;
`exact` computes them in 64 bits, by other steps.  A case is {"op", "way", "dtype", "rows", "cols", "pad"}: `pad` =
elements between the end of a row and the start of the next one; with "top" = alternatives or teacher entries per row, and
for the affine layer "inner" = the input's columns, "act" = the activation, "residual" = whether there is one."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5                # layer norm
TEMPERATURE = 2.0         # distillation


def listed():
    return [
        # one chunk of one stream through a hidden layer: the launch is all there is
        dict(name="ln_fwd_chunk", op="ln", way="forward", dtype="f32", rows=17, cols=768, pad=0),
        # an odd width in half precision, rows that start anywhere
        dict(name="ln_fwd_odd", op="ln", way="forward", dtype="f16", rows=40011, cols=1535, pad=0),
        # long sequences through a wide layer
        dict(name="ln_bwd_wide", op="ln", way="backward", dtype="bf16", rows=32768, cols=4096, pad=0),
        # one chunk of one stream through the output layer: reading the weights is all there is
        dict(name="affine_fwd_chunk", op="affine", way="forward", dtype="f16", rows=17, inner=768, cols=6024, pad=0, act="none", residual=False),
        # 128 utterances of 10 s at a third of the frame rate through a square layer with its bypass
        dict(name="affine_fwd_batch", op="affine", way="forward", dtype="bf16", rows=42752, inner=1536, cols=1536, pad=0, act="relu", residual=True),
        # the derivatives of the output layer for 512 sequences of 50 frames
        dict(name="affine_bwd_output", op="affine", way="backward", dtype="bf16", rows=25600, inner=768, cols=6024, pad=0, act="none", residual=False),
        # one new word over a word list: a single row, with the alternatives that a rescorer keeps
        dict(name="labels_fwd_word", op="labels", way="forward", dtype="f32", rows=1, cols=200003, pad=0, top=8),
        # frame confidences of an alignment: 128 utterances of 10 s over 6024 pdfs
        dict(name="labels_fwd_frames", op="labels", way="forward", dtype="f32", rows=42752, cols=6024, pad=0, top=4),
        # the derivative for a minibatch of sequences over an odd word list
        dict(name="labels_bwd_words", op="labels", way="backward", dtype="bf16", rows=2000, cols=50001, pad=0, top=0),
        # a validation pass over a few utterances in half precision
        dict(name="distill_objf_few", op="distill", way="forward", dtype="f16", rows=300, cols=6024, pad=0, top=10),
        # a student's training minibatch: 128 sequences of 50 frames over 6024 pdfs
        dict(name="distill_train_frames", op="distill", way="train", dtype="f32", rows=6400, cols=6024, pad=0, top=20),
        # a student's training minibatch over a large vocabulary
        dict(name="distill_train_vocab", op="distill", way="train", dtype="bf16", rows=4096, cols=128000, pad=0, top=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op, pad = rng.choice(["ln", "affine", "labels", "distill"]), rng.choice([0, 0, 0, 1, 8])
    if op == "affine":
        inner, cols = _spread(rng, 64, 4096), _spread(rng, 64, 8192)
        if rng.random() < 0.5:  # widths as they are usually chosen
            inner, cols = -(-inner // 64) * 64, -(-cols // 64) * 64
        rows = _spread(rng, 1, min(65536, int(1e11) // (inner * cols)))
        return dict(op=op, way=rng.choice(["forward", "backward"]), dtype=rng.choice(["f16", "bf16"]), rows=rows, inner=inner, cols=cols, pad=pad,
                    act=rng.choice(["none", "relu", "sigmoid", "tanh", "swish", "gelu"]), residual=rng.random() < 0.5)
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "ln":
        cols = _spread(rng, 64, 8192)
        return dict(op=op, way=rng.choice(["forward", "backward"]), dtype=dtype, rows=_spread(rng, 1, (1 << 26) // cols), cols=cols, pad=pad)
    way, cols = rng.choice(["forward", "backward"] if op == "labels" else ["forward", "train"]), _spread(rng, 200, 200000)
    top = 0 if way == "backward" else rng.choice([0, 1, 4, 10, 32]) if op == "labels" else _spread(rng, 1, 128)
    return dict(op=op, way=way, dtype=dtype, rows=_spread(rng, 1, (1 << 27) // cols), cols=cols, pad=pad, top=top)


# ---- inputs

def _matrix(g, rows, cols, pad, dtype, scale=1.0):
    t = torch.empty(rows, cols + pad, dtype=TYPES[dtype], device="cuda")
    t.normal_(0.0, scale, generator=g)
    return t[:, :cols]


def _like(t):
    """a matrix of t's shape, type and row stride, not yet written"""
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rows, cols, pad, dtype, top = case["rows"], case["cols"], case["pad"], case["dtype"], case.get("top", 0)
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    s = {}
    if case["op"] == "ln":
        # activations after an affine layer: every column has its own mean, a few are far from zero
        shift = torch.empty(cols, device="cuda").normal_(0.0, 0.5, generator=g)
        x = _matrix(g, rows, cols, pad, dtype)
        x += shift.to(x.dtype)
        s["x"], s["scale"], s["offset"] = x, 0.5 + rand(cols), rand(cols) - 0.5
        if case["way"] == "backward":
            s["dy"] = _matrix(g, rows, cols, pad, dtype, 0.1)
            xf = x.float()
            s["mean"] = xf.mean(1)
            s["inv_std"] = torch.rsqrt(xf.sub_(s["mean"][:, None]).square_().mean(1) + EPS)
        return s
    if case["op"] == "affine":
        # inputs of unit size (those of a layer norm, or of a ReLU layer), weights that keep it
        s["x"] = _matrix(g, rows, case["inner"], pad, dtype)
        s["weights"] = _matrix(g, cols, case["inner"], pad, dtype, case["inner"] ** -0.5)
        s["bias"] = rand(cols) - 0.5
        if case["way"] == "forward":
            s["residual"] = _matrix(g, rows, cols, pad, dtype) if case["residual"] else None
        else:
            # what the forward pass kept, from which the activation's derivative is taken
            s["pre"] = None if case["act"] == "none" else _matrix(g, rows, cols, pad, dtype)
            s["dy"] = _matrix(g, rows, cols, pad, dtype, 0.1)
        return s
    # a trained network's output: one column per row stands out, more or less
    z = _matrix(g, rows, cols, pad, dtype, 2.0)
    label = (rand(rows) * cols).long().clamp_(max=cols - 1)
    z.scatter_(1, label[:, None], (6.0 + 6.0 * rand(rows, 1)).to(z.dtype))
    s["z"] = z
    if case["op"] == "labels":
        label[rand(rows) < 0.03] = -1  # rows of padding: no label
        s["labels"] = label.to(torch.int32)
        if case["way"] == "backward":
            zf = z.float()
            m = zf.max(1, keepdim=True).values
            d = zf - m
            e = d.exp()
            total = e.sum(1, keepdim=True)
            log_sum = total.log()
            s["stats"] = torch.cat([m, log_sum], 1)
            s["entropy"] = log_sum[:, 0] - (e.mul_(d).sum(1, keepdim=True) / total)[:, 0]
            s["log_prob_deriv"] = rand(rows) - 0.3
            s["entropy_deriv"] = 0.01 * rand(rows)
        return s
    # the teacher's best columns: the one that stands out and others, each row with its own count, some with none
    first = rand(rows, top) * cols
    index = first.long().clamp_(max=cols - 1)
    index[:, 0] = label
    value = (8.0 * rand(rows, 1) + 4.0) - 1.5 * torch.arange(top, device="cuda").float().sqrt() - rand(rows, top)
    count = torch.where(rand(rows) < 0.05, 0.0, (0.5 + 0.5 * rand(rows)) * (top + 1)).long()
    index = torch.where(torch.arange(top, device="cuda")[None, :] < count[:, None], index, -1)
    s["teacher_values"], s["teacher_indexes"] = value.to(z.dtype), index.to(torch.int32)
    s["weights"] = torch.where(rand(rows) < 0.05, 0.0, 0.5 + rand(rows))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    rows, top = case["rows"], case.get("top", 0)
    vector = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
    if case["op"] == "ln":
        if case["way"] == "forward":
            s["y"], s["mean"], s["inv_std"] = _like(s["x"]), vector(rows), vector(rows)
        else:
            s["dx"], s["dscale"], s["doffset"] = _like(s["x"]), vector(case["cols"]), vector(case["cols"])
    elif case["op"] == "affine":
        if case["way"] == "forward":
            s["y"] = torch.empty(rows, case["cols"] + case["pad"], dtype=s["x"].dtype, device="cuda")[:, :case["cols"]]
            s["pre"] = None if case["act"] == "none" else _like(s["y"])
        else:
            s["dx"], s["dweights"], s["dbias"] = _like(s["x"]), _like(s["weights"]), vector(case["cols"])
    elif case["op"] == "labels":
        if case["way"] == "forward":
            s["log_prob"], s["entropy"], s["stats"] = vector(rows), vector(rows), vector(rows, 2)
            s["alt_log_probs"] = vector(rows, top) if top else None
            s["alt_labels"] = torch.empty(rows, top, dtype=torch.int32, device="cuda") if top else None
        else:
            s["dz"] = _like(s["z"])
    else:
        s["objf"] = vector(rows)
        s["dz"] = _like(s["z"]) if case["way"] == "train" else None
    return s


# ---- the package's operators

def _own_ln(s):
    from kaldi_amd import cumatrix
    if s["case"]["way"] == "forward":
        cumatrix.LayerNormPerRow(s["x"], s["scale"], s["offset"], EPS, s["y"], s["mean"], s["inv_std"])
        return s["y"], s["mean"], s["inv_std"]
    cumatrix.DiffLayerNormPerRow(s["x"], s["dy"], s["scale"], s["mean"], s["inv_std"], s["dx"], s["dscale"], s["doffset"])
    return s["dx"], s["dscale"], s["doffset"]


def _own_affine(s):
    from kaldi_amd import cumatrix
    act = s["case"]["act"]
    if s["case"]["way"] == "forward":
        cumatrix.AffinePerRow(s["x"], s["weights"], s["bias"], act, s["residual"], s["y"], s["pre"])
        return s["y"], s["pre"]
    cumatrix.DiffAffinePerRow(s["x"], s["weights"], s["pre"], act, s["dy"], s["dx"], s["dweights"], s["dbias"])
    return s["dx"], s["dweights"], s["dbias"]


def _own_labels(s):
    from kaldi_amd import objective
    if s["case"]["way"] == "forward":
        objective.LabelLogProbs(s["z"], s["labels"], s["log_prob"], s["entropy"], s["stats"], s["alt_log_probs"], s["alt_labels"])
        return [s[k] for k in ("log_prob", "entropy", "stats", "alt_log_probs", "alt_labels")]
    objective.DiffLabelLogProbs(s["z"], s["labels"], s["stats"], s["entropy"], s["log_prob_deriv"], s["entropy_deriv"], s["dz"])
    return s["dz"]


def _own_distill(s):
    from kaldi_amd import objective
    objective.ComputeDistillObjfAndDeriv(objective.DistillationOptions(temperature=TEMPERATURE), s["z"], s["teacher_values"], s["teacher_indexes"],
                                         s["weights"], s["objf"], s["dz"])
    return s["objf"] if s["dz"] is None else (s["objf"], s["dz"])


# ---- their plain form

def _plain_ln(s):
    x = s["x"].float()
    if s["case"]["way"] == "forward":
        mean = x.mean(1, keepdim=True)
        d = x - mean
        inv_std = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
        y = d * inv_std * s["scale"] + s["offset"]
        return y.to(s["x"].dtype), mean[:, 0], inv_std[:, 0]
    dy, inv_std = s["dy"].float(), s["inv_std"][:, None]
    xhat = (x - s["mean"][:, None]) * inv_std
    g = dy * s["scale"]
    dx = inv_std * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)


def _activation(act, z):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "sigmoid":
        return torch.sigmoid(z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "swish":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5))) if act == "gelu" else z


def _slope(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "sigmoid":
        return torch.sigmoid(z) * torch.sigmoid(-z)
    if act == "tanh":
        return 1.0 - torch.tanh(z) ** 2
    if act == "swish":
        return torch.sigmoid(z) * (1.0 + z * torch.sigmoid(-z))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5


def _plain_affine(s):
    act, x, weights, dtype = s["case"]["act"], s["x"].float(), s["weights"].float(), s["x"].dtype
    if s["case"]["way"] == "forward":
        pre = x @ weights.t() + s["bias"]
        y = _activation(act, pre)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(dtype), None if act == "none" else pre.to(dtype)
    dz = s["dy"].float()
    if act != "none":
        dz = dz * _slope(act, s["pre"].float())
    return (dz @ weights).to(dtype), (dz.t() @ x).to(dtype), dz.sum(0)


def _best(z, top):
    """the `top` largest values' columns of every row, largest first, ties to the lowest column: one whole number orders both"""
    bits = (z.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    return ((order << 32) - torch.arange(z.shape[1], device=z.device)).topk(top, 1).indices


def _plain_labels(s):
    z, labels = s["z"].float(), s["labels"].long()
    has = labels >= 0
    at = labels.clamp(min=0)[:, None]
    if s["case"]["way"] == "forward":
        m = z.max(1, keepdim=True).values
        d = z - m
        e = d.exp()
        total = e.sum(1, keepdim=True)
        log_sum = total.log()
        entropy = log_sum - (e * d).sum(1, keepdim=True) / total
        log_prob = torch.where(has, (d.gather(1, at) - log_sum)[:, 0], 0.0)
        out = [log_prob, entropy[:, 0], torch.cat([m, log_sum], 1)]
        if s["case"]["top"]:
            alt = _best(s["z"], s["case"]["top"])
            return out + [d.gather(1, alt) - log_sum, alt.to(torch.int32)]
        return out + [None, None]
    log_q = z - s["stats"][:, :1] - s["stats"][:, 1:]
    q = log_q.exp()
    g = torch.where(has, s["log_prob_deriv"], 0.0)[:, None]
    dz = -g * q - s["entropy_deriv"][:, None] * q * (log_q + s["entropy"][:, None])
    dz.scatter_add_(1, at, g)
    return dz.to(s["z"].dtype)


def _plain_distill(s):
    z, t = s["z"].float() / TEMPERATURE, s["teacher_values"].float() / TEMPERATURE
    index = s["teacher_indexes"].long()
    used = index >= 0
    live = used.any(1, keepdim=True) & (s["weights"] != 0)[:, None]
    at = index.clamp(min=0)
    t = torch.where(used, t, -math.inf)
    e = torch.where(used, (t - t.max(1, keepdim=True).values).exp(), 0.0)
    p = torch.where(used, e / e.sum(1, keepdim=True), 0.0)
    d = z - z.max(1, keepdim=True).values
    ez = d.exp()
    total = ez.sum(1, keepdim=True)
    log_q = d.gather(1, at) - total.log()
    kl = torch.where(p > 0, p * (p.log() - log_q), 0.0).sum(1)
    w = torch.where(live[:, 0], s["weights"], 0.0)
    objf = torch.where(live[:, 0], -w * TEMPERATURE ** 2 * kl, 0.0)
    if s["dz"] is None:
        return objf
    k = (w * TEMPERATURE)[:, None]
    dz = ez * (-k / total)
    dz.scatter_add_(1, at, k * p)
    return objf, dz.to(s["z"].dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ln": _own_ln, "affine": _own_affine, "labels": _own_labels, "distill": _own_distill}[op](state)
    return {"ln": _plain_ln, "affine": _plain_affine, "labels": _plain_labels, "distill": _plain_distill}[op](state)


def work(case):
    n, rows, cols, size, top = case["rows"] * case["cols"], case["rows"], case["cols"], SIZE[case["dtype"]], case.get("top", 0)
    if case["op"] == "ln":
        if case["way"] == "forward":
            return {"bytes": 2 * n * size + 8 * cols + 8 * rows, "flops": 8 * n}
        return {"bytes": 3 * n * size + 12 * cols + 8 * rows, "flops": 14 * n}
    if case["op"] == "affine":
        inner, kept = case["inner"], int(case["act"] != "none")
        if case["way"] == "forward":
            return {"bytes": size * (rows * inner + cols * inner + n * (1 + kept + int(case["residual"]))) + 4 * cols, "flops": 2 * n * inner}
        return {"bytes": size * (2 * rows * inner + 2 * cols * inner + n * (1 + kept)) + 4 * cols, "flops": 4 * n * inner}
    if case["op"] == "labels":
        if case["way"] == "forward":
            return {"bytes": n * size + rows * (4 + 16 + 8 * top), "flops": 6 * n}
        return {"bytes": 2 * n * size + 24 * rows, "flops": 7 * n}
    if case["way"] == "forward":
        return {"bytes": n * size + rows * (8 + top * (size + 4)), "flops": 5 * n}
    return {"bytes": 2 * n * size + rows * (8 + top * (size + 4)), "flops": 6 * n}


# ---- in 64 bits

def _exact_ln(case, s):
    x, scale = s["x"].double(), s["scale"].double()
    if case["way"] == "forward":
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        inv_std = 1.0 / (var + EPS).sqrt()
        return (x - mean) * (inv_std * scale) + s["offset"].double(), mean[:, 0], inv_std[:, 0]
    # with the statistics as they were kept; the row's derivative is that of a projection
    r = s["inv_std"].double()[:, None]
    x.sub_(s["mean"].double()[:, None]).mul_(r)
    dy = s["dy"].double()
    dscale, doffset = torch.einsum("rc,rc->c", dy, x), dy.sum(0)
    dy.mul_(scale)
    along = (dy * x).sum(1, keepdim=True) / case["cols"]
    dy.sub_(dy.sum(1, keepdim=True) / case["cols"]).sub_(x.mul_(along)).mul_(r)
    return dy, dscale, doffset


def _exact_affine(case, s):
    act, x, weights = case["act"], s["x"].double(), s["weights"].double()
    z = torch.addmm(s["bias"].double(), x, weights.t()) if case["way"] == "forward" else None if s["pre"] is None else s["pre"].double()
    if case["way"] == "forward":
        value = {"none": lambda: z, "relu": lambda: torch.relu(z), "sigmoid": lambda: 1.0 / (1.0 + torch.exp(-z)), "tanh": lambda: 1.0 - 2.0 / (torch.exp(2.0 * z) + 1.0),
                 "swish": lambda: z / (1.0 + torch.exp(-z)), "gelu": lambda: z * torch.erfc(-z / math.sqrt(2.0)) / 2.0}[act]()
        return value + s["residual"].double() if case["residual"] else value, None if act == "none" else z
    g = s["dy"].double()
    if act == "relu":
        g[z <= 0] = 0.0
    elif act in ("sigmoid", "tanh"):
        g /= (2.0 * torch.cosh(z / 2.0)) ** 2 if act == "sigmoid" else torch.cosh(z) ** 2
    elif act == "swish":
        g *= 1.0 / (1.0 + torch.exp(-z)) + z / (2.0 * torch.cosh(z / 2.0)) ** 2
    elif act == "gelu":
        g *= torch.erfc(-z / math.sqrt(2.0)) / 2.0 + z * torch.exp(-z.square() / 2.0) / math.sqrt(2.0 * math.pi)
    return torch.mm(g, weights), torch.mm(x.t(), g).t(), g.sum(0)


def _exact_labels(case, s):
    z, labels = s["z"].double(), s["labels"].long()
    at = torch.arange(case["rows"], device="cuda")
    if case["way"] == "forward":
        log_z = torch.logsumexp(z, 1)
        m = z.amax(1)
        lp = torch.where(labels >= 0, z[at, labels.clamp(min=0)] - log_z, 0.0)
        best = z.topk(case["top"], 1).values - log_z[:, None] if case["top"] else None
        z.sub_(log_z[:, None])
        entropy = -(z.exp() * z).sum(1)
        return [lp, entropy, torch.stack([m, log_z - m], 1), best, None]
    z.sub_(s["stats"].double().sum(1, keepdim=True))
    q = z.exp()
    g = torch.where(labels >= 0, s["log_prob_deriv"].double(), 0.0)
    z.add_(s["entropy"].double()[:, None]).mul_(s["entropy_deriv"].double()[:, None]).add_(g[:, None]).mul_(q).neg_()
    z[at, labels.clamp(min=0)] += g
    return z


def _exact_distill(case, s):
    z, index = s["z"].double().div_(TEMPERATURE), s["teacher_indexes"].long()
    used = index >= 0
    t = (s["teacher_values"].double() / TEMPERATURE).masked_fill(~used, -1e300)
    log_p = t - torch.logsumexp(t, 1, keepdim=True)
    p = log_p.exp() * used
    live = used.any(1)
    w = s["weights"].double() * live
    log_z = torch.logsumexp(z, 1, keepdim=True)
    log_q = z.gather(1, index.clamp(min=0)) - log_z
    objf = TEMPERATURE ** 2 * w * ((log_q - log_p) * p).masked_fill(~used, 0.0).sum(1)
    if case["way"] == "forward":
        return objf
    z.sub_(log_z).exp_().neg_().scatter_add_(1, index.clamp(min=0), p).mul_((TEMPERATURE * w)[:, None])
    return objf, z


def exact(case, seed):
    s = _inputs(case, seed)
    return {"ln": _exact_ln, "affine": _exact_affine, "labels": _exact_labels, "distill": _exact_distill}[case["op"]](case, s)
