"""Operators that surround the recurrent layers of a language model, as cases to be measured and compared:

* the gated linear recurrence  f = sigmoid(g + b),  c_t = f_t c_{t-1} + (1 - f_t) x_t,  h_t = c_t  (0 at padded positions,
  where the state is carried), over (length, batch, 2 * hidden) tensors whose last dimension holds the pairs (x, g);
* the scaled embedding lookup  y_n = scale * W[token_n]  and its gradient  dW[v] = scale * sum over {n: token_n = v} of dy_n;
* the orthogonalised update: X_0 = G / (|G|_F + eps), then five times X <- (a I + b X X^T + c (X X^T)^2) X.

``run`` computes a case with elementary torch operations in 32 bits or, where ``own`` is true, through this package.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


# ---------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------
def recurrence(name, length, batch, hidden, dtype, train, mask=False, reverse=False, bias=True, init=True):
    return {"name": name, "op": "recurrence", "length": length, "batch": batch, "hidden": hidden, "dtype": dtype,
            "train": train, "mask": mask, "reverse": reverse, "bias": bias, "init": init}


def embedding(name, tokens, vocabulary, hidden, table, out, train, flat=False, padding=False):
    return {"name": name, "op": "embedding", "tokens": tokens, "vocabulary": vocabulary, "hidden": hidden, "table": table,
            "out": out, "train": train, "flat": flat, "padding": padding}


def update(name, batch, rows, cols, dtype, out):
    return {"name": name, "op": "update", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype, "out": out}


def listed():
    return [
        # one new token for each of 64 sequences of the hidden-2048 language model: latency
        recurrence("recurrence_token", 1, 64, 2048, "bfloat16", False),
        # long-sequence inference, 16 documents of 8192 tokens
        recurrence("recurrence_documents", 8192, 16, 1024, "bfloat16", False, init=False),
        # one sequence of 65536 tokens: few columns, all the parallelism is along time
        recurrence("recurrence_one_long", 65536, 1, 2048, "bfloat16", False),
        # a training step's layer of the hidden-2048 language model, state handed on from the previous segment
        recurrence("recurrence_train_lm", 512, 32, 2048, "float16", True),
        # the backward direction of a speech layer, padded sequences
        recurrence("recurrence_train_speech", 1000, 24, 1024, "bfloat16", True, mask=True, reverse=True, init=False),
        # a small float32 model with sizes that fit no vector
        recurrence("recurrence_train_odd", 777, 5, 201, "float32", True, mask=True),
        # the tokens of one decoding step of 64 sequences
        embedding("embedding_token", 64, 50000, 2048, "bfloat16", "bfloat16", False),
        # the input of a training step: 512 x 32 word-frequency tokens, float32 master table, 16-bit activations
        embedding("embedding_train_words", 16384, 50000, 2048, "float32", "bfloat16", True, padding=True),
        # byte-level text: 205 symbols, each of them hundreds of times
        embedding("embedding_train_bytes", 32768, 205, 520, "float32", "float32", True),
        # the projection of a hidden-128 layer: latency
        update("update_small", 1, 128, 384, "float32", "bfloat16"),
        # the down-projections of the six layers of the language model, taller than wide, one call
        update("update_six_layers", 6, 2048, 512, "float32", "bfloat16"),
        # the projection of a bidirectional hidden-1024 layer
        update("update_large", 1, 2048, 6144, "bfloat16", "bfloat16"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread evenly over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["token", "prompt", "train", "lookup", "table", "update"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    whole = rng.choice([1, 1, 8, 64])               # multiples of 8 and 64 are what models have; the others are odd

    def size(low, high):
        n = _spread(rng, low, high)
        return max(whole * math.ceil(low / whole), n // whole * whole)

    if op == "token":
        c = recurrence("", 1, _spread(rng, 1, 256), size(16, 4096), dtype, False, bias=rng.random() < 0.7,
                       mask=rng.random() < 0.2)
    elif op in ("prompt", "train"):
        most = 2 ** 27 if op == "prompt" else 2 ** 25   # elements of one (length, batch, hidden) tensor
        if dtype == "float32":
            most //= 2
        hidden = size(16, 4096)
        length = _spread(rng, 2, 65536 if op == "prompt" else 8192)
        batch = _spread(rng, 1, max(1, min(256, most // (hidden * length))))
        length = max(1, min(length, most // (hidden * batch)))
        c = recurrence("", length, batch, hidden, dtype, op == "train", mask=rng.random() < 0.4,
                       reverse=rng.random() < 0.3, bias=rng.random() < 0.7, init=rng.random() < 0.6)
    elif op in ("lookup", "table"):
        hidden = size(8, 2048)
        tokens = _spread(rng, 1, 4096) if op == "lookup" else _spread(rng, 64, 65536)
        tokens = min(tokens, 16384 * 2048 // hidden)
        vocabulary = _spread(rng, 100, min(200000, 50000 * 2048 // hidden))
        out = rng.choice(["float16", "bfloat16", dtype]) if dtype == "float32" else dtype
        c = embedding("", tokens, vocabulary, hidden, dtype, out, op == "table", flat=rng.random() < 0.3,
                      padding=rng.random() < 0.4)
    else:
        rows, cols = size(8, 2048), size(8, 6144)
        if rng.random() < 0.4:
            rows, cols = cols, rows
        small = min(rows, cols)
        most = 2048 * 2048 * 6144                    # products of the largest listed case
        batch = _spread(rng, 1, max(1, min(12, most // (small * rows * cols))))
        c = update("", batch, rows, cols, dtype, "bfloat16" if dtype == "float32" else dtype)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "recurrence":
        L, B, d, dt = case["length"], case["batch"], case["hidden"], DTYPES[case["dtype"]]
        u = _normal(g, L, B, 2 * d, dtype=dt)
        # forget biases of layers that remember tens to hundreds of steps
        bias = torch.rand(d, generator=g, device="cuda") * 4.0 + 1.0 if case["bias"] else None
        c0 = _normal(g, B, d) * 0.3 if case["init"] else None
        mask = None
        if case["mask"]:
            # lengths from 60 % of the longest on, the tail is padding; a batch of several has an empty sequence as well
            lengths = (torch.rand(B, generator=g, device="cuda") * 0.4 + 0.6).mul(L).ceil().long()
            if B > 2:
                lengths[B // 2] = 0
            mask = torch.arange(L, device="cuda").view(L, 1) >= lengths.view(1, B)
        state = {"case": case, "u": u, "bias": bias, "c0": c0, "mask": mask}
        if case["train"]:
            state["grad_h"] = _normal(g, L, B, d, dtype=dt)
            state["grad_last"] = _normal(g, B, d)
            for k in ("u", "bias", "c0"):
                if state[k] is not None:
                    state[k].requires_grad_()
        elif L == 1:
            state["u"] = u[0]                       # the (batch, features) form of a single token
            if mask is not None:
                state["mask"] = mask[0]
        return state
    if case["op"] == "embedding":
        n, v, d = case["tokens"], case["vocabulary"], case["hidden"]
        table = _normal(g, v, d, dtype=DTYPES[case["table"]])
        # word frequencies fall off with the rank; ``flat``: every token as likely as any other
        if case["flat"]:
            rank = torch.randint(0, v, (n,), generator=g, device="cuda")
        else:
            rank = (torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        order = torch.randperm(v, generator=g, device="cuda")
        tokens = order[rank]
        padding = None
        if case["padding"]:
            padding = v // 3                       # a tenth of the positions is padding
            tokens[torch.rand(n, generator=g, device="cuda") < 0.1] = padding
        state = {"case": case, "table": table, "tokens": tokens, "padding": padding, "scale": math.sqrt(d)}
        if case["train"]:
            state["grad"] = _normal(g, n, d, dtype=DTYPES[case["out"]])
            table.requires_grad_()
        return state
    k, m, n = case["batch"], case["rows"], case["cols"]
    # momentum of a weight: a few strong directions over noise
    strong = _normal(g, k, m, 16) @ _normal(g, k, 16, n) * 0.25
    grad = ((strong + _normal(g, k, m, n)) * 1e-3).to(DTYPES[case["dtype"]])
    return {"case": case, "grad": grad if k > 1 else grad[0]}


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def _scan(a, b):
    """Every prefix of y_t = a_t y_{t-1} + b_t (y before the first is 0) along the first dimension, by doubling."""
    step, length = 1, a.size(0)
    while step < length:
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_recurrence(s):
    case = s["case"]
    u, bias, c0, mask = (None if s[k] is None else s[k].detach() for k in ("u", "bias", "c0", "mask"))
    single = u.dim() == 2
    if single:
        u = u.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    length, batch = u.shape[:2]
    pairs = u.float().view(length, batch, -1, 2)
    if case["reverse"]:
        pairs = pairs.flip(0)
        mask = None if mask is None else mask.flip(0)
    x, gate = pairs[..., 0], pairs[..., 1]
    if bias is not None:
        gate = gate + bias.float()
    f, keep = torch.sigmoid(gate), torch.sigmoid(-gate)          # keep = 1 - f without cancellation
    add = keep * x
    zero = torch.zeros((), device=u.device)
    if mask is not None:
        pad = mask.unsqueeze(-1)
        f, add = torch.where(pad, zero + 1.0, f), torch.where(pad, zero, add)
    first = torch.zeros(batch, x.size(2), device=u.device) if c0 is None else c0.float()
    c = _scan(f, torch.cat([add[:1] + f[:1] * first, add[1:]]))
    h = c if mask is None else torch.where(pad, zero, c)
    out_h = (h.flip(0) if case["reverse"] else h).to(u.dtype)
    last = c[-1].clone()
    if not case["train"]:
        return {"h": out_h[0] if single else out_h, "c_last": last}
    grad = s["grad_h"].float()
    if case["reverse"]:
        grad = grad.flip(0)
    if mask is not None:
        grad = torch.where(pad, zero, grad)
    grad = torch.cat([grad[:-1], grad[-1:] + s["grad_last"]])
    # dc_t = grad_t + f_{t+1} dc_{t+1}: the same recurrence, backwards in time
    follow = torch.cat([f[1:], torch.ones_like(f[:1])]).flip(0)
    dc = _scan(follow, grad.flip(0)).flip(0)
    before = torch.cat([first.unsqueeze(0), c[:-1]])
    dx, dgate = dc * keep, dc * (before - x) * f * keep
    if mask is not None:
        dx, dgate = torch.where(pad, zero, dx), torch.where(pad, zero, dgate)
    du = torch.stack([dx, dgate], dim=-1).view(length, batch, -1)
    out = {"h": out_h, "c_last": last, "grad_u": (du.flip(0) if case["reverse"] else du).to(u.dtype)}
    if bias is not None:
        out["grad_bias"] = dgate.sum((0, 1))
    if c0 is not None:
        out["grad_c0"] = dc[0] * f[0]
    return out


def _plain_embedding(s):
    case, table, tokens = s["case"], s["table"].detach(), s["tokens"]
    out = {"y": (table[tokens].float() * s["scale"]).to(DTYPES[case["out"]])}
    if case["train"]:
        dy = s["grad"].float() * s["scale"]
        if s["padding"] is not None:
            dy = torch.where((tokens == s["padding"]).unsqueeze(1), torch.zeros((), device=dy.device), dy)
        total = torch.zeros(table.shape, device=table.device)
        out["grad_table"] = total.index_add_(0, tokens, dy).to(table.dtype)
    return out


def _plain_update(s):
    a, b, c = COEFFICIENTS
    g = s["grad"].float()
    tall = g.size(-2) > g.size(-1)
    x = g.transpose(-1, -2) if tall else g
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(-1, -2) if tall else x).to(DTYPES[s["case"]["out"]]).contiguous()


def _own_recurrence(s):
    from sru_b200.linear_recurrence import gated_linear_recurrence
    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            h, last = gated_linear_recurrence(s["u"], s["c0"], s["bias"], s["mask"], reverse=case["reverse"])
        return {"h": h, "c_last": last}
    h, last = gated_linear_recurrence(s["u"], s["c0"], s["bias"], s["mask"], reverse=case["reverse"])
    leaves = {k: s[k] for k in ("u", "bias", "c0") if s[k] is not None}
    grads = torch.autograd.grad((h, last), list(leaves.values()), (s["grad_h"], s["grad_last"]))
    return {"h": h.detach(), "c_last": last.detach(), **{"grad_" + k: v for k, v in zip(leaves, grads)}}


def _own_embedding(s):
    from sru_b200.embedding import embedding_lookup
    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            return {"y": embedding_lookup(s["tokens"], s["table"], scale=s["scale"], padding_idx=s["padding"],
                                          out_dtype=DTYPES[case["out"]])}
    y = embedding_lookup(s["tokens"], s["table"], scale=s["scale"], padding_idx=s["padding"], out_dtype=DTYPES[case["out"]])
    (grad,) = torch.autograd.grad(y, s["table"], s["grad"])
    return {"y": y.detach(), "grad_table": grad}


def _own_update(s):
    from sru_b200.orthogonalize import orthogonalize
    return orthogonalize(s["grad"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, out_dtype=DTYPES[s["case"]["out"]])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"recurrence": _own_recurrence, "embedding": _own_embedding, "update": _own_update}[op](state)
    return {"recurrence": _plain_recurrence, "embedding": _plain_embedding, "update": _plain_update}[op](state)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "recurrence":
        L, B, d, s = case["length"], case["batch"], case["hidden"], SIZE[case["dtype"]]
        n, columns = L * B * d, B * d
        small = 4 * columns * (2 if case["init"] else 1) + (4 * d if case["bias"] else 0) + (L * B if case["mask"] else 0)
        bytes_, flops = n * 3 * s + small, 12 * n      # u in, h out
        if case["train"]:                              # grad_h in, grad_u out
            bytes_ += n * 3 * s + 4 * columns * (2 if case["init"] else 1) + (4 * d if case["bias"] else 0)
            flops += 16 * n
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "embedding":
        n, v, d = case["tokens"], case["vocabulary"], case["hidden"]
        rows = min(n, v)                               # a row of the table is read once however often it is asked for
        bytes_ = 8 * n + rows * d * SIZE[case["table"]] + n * d * SIZE[case["out"]]
        if case["train"]:
            bytes_ += n * d * SIZE[case["out"]] + v * d * SIZE[case["table"]]
        return {"bytes": bytes_, "flops": n * d * (3 if case["train"] else 1)}
    k, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # X X^T and its square are symmetric: half of each product
    return {"bytes": k * m * n * (SIZE[case["dtype"]] + SIZE[case["out"]]),
            "flops": k * STEPS * (m * m * n + m ** 3 + 2 * m * m * n)}


# ---------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_recurrence(s):
    """Step by step in time; the backward pass walks the chain rule the other way."""
    case = s["case"]
    u = s["u"].detach().double()
    mask = s["mask"]
    single = u.dim() == 2
    if single:
        u = u.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    length, batch, width = u.shape
    d = width // 2
    bias = 0.0 if s["bias"] is None else s["bias"].detach().double()
    c = torch.zeros(batch, d, dtype=torch.float64, device=u.device) if s["c0"] is None else s["c0"].detach().double()
    times = range(length - 1, -1, -1) if case["reverse"] else range(length)
    train = case["train"]
    h = torch.empty(length, batch, d, dtype=torch.float64, device=u.device)
    history = torch.empty_like(h) if train else None
    for t in times:
        f = torch.sigmoid(u[t, :, 1::2] + bias)
        new = torch.lerp(u[t, :, 0::2], c, f)
        if train:
            history[t] = c
        if mask is None:
            c = new
            h[t] = c
        else:
            live = ~mask[t].unsqueeze(1)
            c = torch.where(live, new, c)
            h[t] = torch.where(live, c, torch.zeros_like(c))
    out = {"h": h[0] if single else h, "c_last": c}
    if not train:
        return out
    dc = s["grad_last"].double()
    du = torch.zeros_like(u)
    dbias = torch.zeros(d, dtype=torch.float64, device=u.device)
    for t in reversed(times):
        f = torch.sigmoid(u[t, :, 1::2] + bias)
        total = dc + s["grad_h"][t].double()
        dx = total * (1.0 - f)
        dg = total * (history[t] - u[t, :, 0::2]) * f * (1.0 - f)
        before = total * f
        if mask is not None:
            live = ~mask[t].unsqueeze(1)
            zero = torch.zeros_like(dx)
            dx, dg, before = torch.where(live, dx, zero), torch.where(live, dg, zero), torch.where(live, before, dc)
        du[t, :, 0::2], du[t, :, 1::2] = dx, dg
        dbias += dg.sum(0)
        dc = before
    out["grad_u"] = du
    if s["bias"] is not None:
        out["grad_bias"] = dbias
    if s["c0"] is not None:
        out["grad_c0"] = dc
    return out


def _exact_embedding(s):
    case, tokens = s["case"], s["tokens"]
    table = s["table"].detach().double()
    out = {"y": torch.index_select(table, 0, tokens) * s["scale"]}
    if case["train"]:
        # sums over runs of equal tokens as differences of running totals in 64 bits
        order = torch.argsort(tokens, stable=True)
        dy = s["grad"].double()[order] * s["scale"]
        counts = torch.bincount(tokens, minlength=table.size(0))
        ends = counts.cumsum(0)
        totals = torch.cat([torch.zeros(1, dy.size(1), dtype=torch.float64, device=dy.device), dy.cumsum(0)])
        grad = totals[ends] - totals[ends - counts]
        if s["padding"] is not None:
            grad[s["padding"]] = 0.0
        out["grad_table"] = grad
    return out


def _exact_update(s):
    """The steps act on the singular values alone: X = p(G G^T / (|G| + eps)^2) G / (|G| + eps), p taken at the
    eigenvalues of the smaller Gram matrix."""
    a, b, c = COEFFICIENTS
    g = s["grad"].double()
    tall = g.size(-2) > g.size(-1)
    x = g.mT if tall else g
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
    values, vectors = torch.linalg.eigh(x @ x.mT)
    lam, factor = values.clamp_min(0.0), torch.ones_like(values)
    for _ in range(STEPS):
        gain = a + b * lam + c * lam * lam
        factor, lam = factor * gain, lam * gain * gain
    x = (vectors * factor.unsqueeze(-2)) @ (vectors.mT @ x)
    return x.mT.contiguous() if tall else x


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "embedding": _exact_embedding, "update": _exact_update}[case["op"]](state)
