"""What the operators that learn node classifiers are measured on.

Four operators, as stag_amd.train offers them: the scores of packed one-hot rows against a table of coefficients (an embedding
lookup summed over a row's tokens), the gradient of that table, the logistic loss of siblings with its gradient, and an AdamW
step over many tensors.  Sizes are those of the package's own workloads: 16S alignments (1,500 columns, 7,500 features), protein
marker genes (1,050 columns), concatenated marker genes (31,500 columns), and fan-outs and level widths of their trees.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256          # values that share a scale in 8-bit optimizer states; every tensor's state begins at a multiple of it
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one read scored against the children of one node: what an interactive query waits for
        {"name": "scores one read", "op": "scores", "m": 1, "ncol": 1500, "k": 8, "type": "f32", "indexed": False},
        # one training batch at one node (13 children), rows picked out of the training set, the last ones padding
        {"name": "scores node batch", "op": "scores", "m": 4096, "ncol": 1500, "k": 13, "type": "f32", "indexed": True},
        # all classifiers of a level of the 16S tree at once
        {"name": "scores level", "op": "scores", "m": 8192, "ncol": 1500, "k": 1000, "type": "f32", "indexed": True},
        # genomes: rows of concatenated marker genes, table in 16 bits
        {"name": "scores genomes bf16", "op": "scores", "m": 2000, "ncol": 31500, "k": 40, "type": "bf16", "indexed": False},
        # a node with few training sequences, protein marker gene
        {"name": "grad small node", "op": "grad", "m": 64, "ncol": 1050, "k": 4, "type": "f32", "indexed": False},
        {"name": "grad node batch", "op": "grad", "m": 4096, "ncol": 1500, "k": 13, "type": "f32", "indexed": True},
        {"name": "grad level bf16", "op": "grad", "m": 8192, "ncol": 1500, "k": 1000, "type": "bf16", "indexed": True},
        # the loss of one node's batch, and of a level where a row trains only the siblings of its place
        {"name": "loss node", "op": "loss", "m": 300, "k": 8, "type": "f32", "siblings": False},
        {"name": "loss level", "op": "loss", "m": 65536, "k": 1000, "type": "bf16", "siblings": True},
        # the step of one node's table and bias, of a whole tree's, and of a tree's with 8-bit states and 16-bit tables
        {"name": "adamw node", "op": "adamw", "tables": 1, "ncol": 1500, "fanout": 8, "type": "f32", "bits": 32},
        {"name": "adamw tree", "op": "adamw", "tables": 1600, "ncol": 1500, "fanout": 4, "type": "f32", "bits": 32},
        {"name": "adamw tree 8 bit", "op": "adamw", "tables": 1600, "ncol": 1500, "fanout": 4, "type": "bf16", "bits": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["scores", "scores", "grad", "grad", "loss", "adamw"])
    kind = rng.choice(["f32", "f32", "bf16", "f16"])
    if op in ("scores", "grad"):
        m, ncol = _log(rng, 1, 8192), rng.choice([_log(rng, 29, 1500), _log(rng, 29, 1500), _log(rng, 1500, 31500)])
        most = 8192 * 1500 * 1000 // (m * ncol)
        if ncol > 1500:                    # the wide rows of genomes come in smaller batches
            m = min(m, 2000)
            most = 2000 * 31500 * 40 // (m * ncol)
        return {"op": op, "m": m, "ncol": ncol, "k": _log(rng, 1, max(1, min(1000, most))), "type": kind, "indexed": rng.random() < 0.5}
    if op == "loss":
        m = _log(rng, 1, 65536)
        return {"op": op, "m": m, "k": _log(rng, 1, min(4000, 65536 * 1000 // m)), "type": kind, "siblings": rng.random() < 0.6}
    ncol, fanout = _log(rng, 29, 1500), _log(rng, 1, 40)
    return {"op": op, "tables": _log(rng, 1, max(1, min(1600, 1600 * 1500 * 4 // (ncol * fanout)))), "ncol": ncol, "fanout": fanout, "type": kind, "bits": rng.choice([8, 32])}


def _words(n_features):
    return -(-n_features // 128) * 4       # packed rows are whole 16-byte units


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _packed_rows(g, n, ncol, classes):
    """n packed one-hot rows: sequences that differ from the consensus of their class in 5 % of the columns, 3 % of them gaps."""
    consensus = torch.randint(1, 5, (classes, ncol), generator=g, device=DEV, dtype=torch.int8)
    which = torch.randint(0, classes, (n,), generator=g, device=DEV)
    words = _words(5 * ncol)
    bits = torch.empty((n, words), dtype=torch.int32, device=DEV)
    shift = torch.arange(32, device=DEV, dtype=torch.int64)
    step = max(1, (1 << 26) // (32 * words))
    for a in range(0, n, step):
        sym = consensus[which[a:a + step]]
        u = torch.rand(sym.shape, generator=g, device=DEV)
        other = torch.randint(1, 5, sym.shape, generator=g, device=DEV, dtype=torch.int8)
        sym = torch.where(u < 0.05, other, torch.where(u < 0.08, torch.zeros_like(sym), sym)).to(torch.int64)
        onehot = torch.zeros((sym.shape[0], 32 * words), dtype=torch.int64, device=DEV)
        onehot.scatter_(1, sym + 5 * torch.arange(ncol, device=DEV), 1)
        bits[a:a + step] = (onehot.view(sym.shape[0], words, 32) << shift).sum(-1).to(torch.int32)
    return bits, which


def _prepare_rows(case, seed):
    g = _gen(seed)
    m, ncol, k = case["m"], case["ncol"], case["k"]
    n = m + m // 2 + 1 if case["indexed"] else m
    bits, _ = _packed_rows(g, n, ncol, 16)
    rows = None
    if case["indexed"]:
        rows = torch.randint(0, n, (m,), generator=g, device=DEV, dtype=torch.int32)
        if m >= 16:
            rows[m - m // 16:] = -1        # the batch is padded to its size
    s = {"bits": bits, "rows": rows, "scale": 1.0 / math.sqrt(ncol), "n_features": 5 * ncol}
    kind = DTYPES[case["type"]]
    if case["op"] == "scores":
        w = torch.randn((5 * ncol, k), generator=g, device=DEV)
        s["table"] = (w * (torch.rand(w.shape, generator=g, device=DEV) < 0.3)).to(kind)     # LASSO: many coefficients are zero
        s["bias"] = torch.randn((k,), generator=g, device=DEV)
    else:
        u = torch.rand((m, k), generator=g, device=DEV)
        sign = torch.where(torch.rand((m, k), generator=g, device=DEV) < 0.3, -1.0, 1.0)
        s["grad"] = (sign * u * u).to(kind)              # sigmoid minus target: many near zero
    return s


def _prepare_loss(case, seed):
    g = _gen(seed)
    m, k = case["m"], case["k"]
    s = {"scores": 3.0 * torch.randn((m, k), generator=g, device=DEV), "scale": 1.0 / m, "kind": DTYPES[case["type"]]}
    s["weight"] = 0.5 + torch.rand((m,), generator=g, device=DEV)
    if case["siblings"]:                   # groups of siblings: children of one node are neighbours
        cuts = torch.cat([torch.zeros(1, device=DEV), (torch.rand((k,), generator=g, device=DEV) < 0.25).float()])[:k]
        first = torch.nonzero(cuts > 0).flatten().to(torch.int32)
        first = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), first])
        last = torch.cat([first[1:], torch.full((1,), k, dtype=torch.int32, device=DEV)])
        group = torch.randint(0, first.numel(), (m,), generator=g, device=DEV)
        lo, hi = first[group], last[group]
        hi = torch.where(torch.rand((m,), generator=g, device=DEV) < 0.05, lo, hi)           # rows that train nothing here
        s["siblings"] = torch.stack([lo, hi], 1).contiguous()
    else:
        lo, hi = torch.zeros((m,), dtype=torch.int32, device=DEV), torch.full((m,), k, dtype=torch.int32, device=DEV)
        s["siblings"] = None
    label = lo + (torch.rand((m,), generator=g, device=DEV) * (hi - lo)).to(torch.int32)
    s["label"] = torch.where((torch.rand((m,), generator=g, device=DEV) < 0.1) | (hi <= lo), -1, torch.minimum(label, (hi - 1).clamp(min=0))).to(torch.int32)
    return s


def _fanouts(case):
    """Children of each node: around the mean, the same for every seed (they are a tree's, not an input's)."""
    return [max(1, (case["fanout"] * (1 + (37 * i) % 8)) // 4) if case["tables"] > 1 else case["fanout"] for i in range(case["tables"])]


def _shapes(case):
    f = 5 * case["ncol"]
    return [shape for k in _fanouts(case) for shape in ((f, k), (k,))]


def _prepare_adamw(case, seed):
    g = _gen(seed)
    shapes, starts, at = _shapes(case), [], 0
    for shape in shapes:
        starts.append(at)
        at += -(-math.prod(shape) // BLOCK) * BLOCK
    kind = DTYPES[case["type"]]
    real = torch.zeros(at, dtype=torch.bool, device=DEV)
    for start, shape in zip(starts, shapes):
        real[start:start + math.prod(shape)] = True

    def values(make):
        return torch.where(real, make(), 0.0)

    flat = values(lambda: 0.1 * torch.randn(at, generator=g, device=DEV)).to(kind)
    spread = torch.exp(2.0 * torch.randn(at, generator=g, device=DEV))           # gradients differ by orders of magnitude
    grad = values(lambda: 1e-3 * spread * torch.randn(at, generator=g, device=DEV)).to(kind)
    m = values(lambda: 4e-4 * spread * torch.randn(at, generator=g, device=DEV))
    v = values(lambda: (1e-3 * spread * (0.5 + torch.rand(at, generator=g, device=DEV))) ** 2)
    s = {"flat": flat, "grad": grad, "step": 40, "lr": 1e-3, "m": m, "v": v}
    if case["bits"] == 8:
        s["m_scale"], s["v_scale"] = _scale_of(m), _scale_of(v.sqrt())
        s["m"] = _nearest(m, s["m_scale"])
        s["v"] = _nearest(v.sqrt(), s["v_scale"])
    decay = [(0.01, 1e-4) if len(shape) == 2 else (0.0, 0.0) for shape in shapes]            # biases are not penalised
    of_block = torch.tensor([n for n, shape in enumerate(shapes) for _ in range(-(-math.prod(shape) // BLOCK))], device=DEV)
    s["decay"] = torch.tensor([d[0] for d in decay], device=DEV)[of_block].unsqueeze(1)
    s["l1"] = torch.tensor([d[1] for d in decay], device=DEV)[of_block].unsqueeze(1)
    if own:                                # the optimizer a program keeps: it holds parameters, gradients and states
        from stag_amd import train
        views = [flat[a:a + math.prod(shape)].view(shape) for a, shape in zip(starts, shapes)]
        grads = [grad[a:a + math.prod(shape)].view(shape) for a, shape in zip(starts, shapes)]
        s["opt"] = train.AdamW(views, grads, lr=s["lr"], betas=(BETA1, BETA2), eps=EPS, weight_decay=[d[0] for d in decay],
                               l1=[d[1] for d in decay], state_bits=case["bits"])
        s["opt"].load_state(s["step"], s["m"], s["v"], s.get("m_scale"), s.get("v_scale"))
    return s


def _scale_of(x):
    """The smallest power of two s with max|x| <= 448 s in each block of 256."""
    top = x.view(-1, BLOCK).abs().amax(1).clamp(min=2.0 ** -117)
    mant, exp = torch.frexp(top)           # top = mant * 2^exp, 0.5 <= mant < 1; 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(top), exp - 9 + (mant > 0.875).to(exp.dtype))


def _nearest(x, scale):
    return (x.view(-1, BLOCK) / scale.unsqueeze(1)).to(torch.float8_e4m3fn).flatten()


def prepare(case, seed):
    return {"case": case, **{"scores": _prepare_rows, "grad": _prepare_rows, "loss": _prepare_loss, "adamw": _prepare_adamw}[case["op"]](case, seed)}


# ---------------------------------------------------------------------------------------------------------------- passes
def _unpacked(s, kind):
    """The batch's rows as zeros and ones, padding rows as zeros, and which rows are no padding."""
    bits, rows = s["bits"], s["rows"]
    real = None
    if rows is not None:
        real = (rows >= 0) & (rows < bits.shape[0])
        bits = bits[torch.where(real, rows, 0).long()]
    x = ((bits.unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).view(bits.shape[0], -1)[:, :s["n_features"]].to(kind)
    return (x if real is None else x * real.unsqueeze(1).to(kind)), real


def _plain_scores(s):
    x, real = _unpacked(s, torch.float32)
    out = (x @ s["table"].float()) * s["scale"] + s["bias"]
    return out if real is None else torch.where(real.unsqueeze(1), out, 0.0)


def _plain_grad(s):
    x, real = _unpacked(s, torch.float32)
    grad = s["grad"].float()
    if real is not None:
        grad = torch.where(real.unsqueeze(1), grad, 0.0)
    return (x.t() @ grad) * s["scale"], grad.double().sum(0).float()


def _plain_loss(s):
    scores, label = s["scores"], s["label"].unsqueeze(1)
    column = torch.arange(scores.shape[1], device=DEV, dtype=torch.int32)
    y = column == label
    z = torch.where(y, -scores, scores)
    e = torch.exp(-z.abs())
    weight = (s["weight"] * s["scale"]).unsqueeze(1)
    loss = (z.clamp(min=0) + torch.log1p(e)) * weight
    p = torch.where(z >= 0, 1.0, e) / (1.0 + e) * weight
    grad = torch.where(y, -p, p)
    if s["siblings"] is not None:
        inside = (column >= s["siblings"][:, :1]) & (column < s["siblings"][:, 1:])
        loss, grad = torch.where(inside, loss, 0.0), torch.where(inside, grad, 0.0)
    return loss.double().sum(0).float(), grad.to(s["kind"])


def _mix(at, step):
    """16 + 16 bits for each position: a 32-bit integer hash (two rounds of shift, exclusive or and multiply)."""
    x = (at ^ (step * 0x9E3779B9)) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    return x >> 16, x & 0xFFFF


def _rounded(x, scale, chance):
    """x / scale in e4m3, up or down by `chance` (16 bits): on the mean the value itself."""
    y = x / scale
    a = y.abs()
    bits = (a.view(torch.int32) + ((chance << 4) | 8).to(torch.int32)) & -(1 << 20)
    small = torch.floor(a * 512.0 + (chance.float() + 0.5) * (2.0 ** -16)) * (2.0 ** -9)     # below 2^-6 codes are 2^-9 apart
    return torch.copysign(torch.where(a < 2.0 ** -6, small, bits.view(torch.float32)), y).to(torch.float8_e4m3fn)


def _plain_adamw(s):
    s["step"] += 1
    t, lr = s["step"], s["lr"]
    c1, c2 = lr / (1.0 - BETA1 ** t), 1.0 / math.sqrt(1.0 - BETA2 ** t)
    g = s["grad"].float().view(-1, BLOCK)
    small = s["m"].dtype == torch.float8_e4m3fn
    m, v = s["m"].float().view(-1, BLOCK), s["v"].float().view(-1, BLOCK)
    if small:
        m, v = m * s["m_scale"].unsqueeze(1), v * s["v_scale"].unsqueeze(1)
        v = v * v
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = v.sqrt()
    d = root * c2 + EPS
    p = s["flat"].float().view(-1, BLOCK)
    p = p * (1.0 - lr * s["decay"]) - c1 * m / d
    p = torch.sign(p) * (p.abs() - lr * s["l1"] / d).clamp(min=0)
    s["flat"].copy_(p.flatten())
    if not small:
        s["m"].copy_(m.flatten())
        s["v"].copy_(v.flatten())
        return s["flat"], s["m"], s["v"]
    hi, lo = _mix(torch.arange(g.numel(), device=DEV, dtype=torch.int64).view(-1, BLOCK), t)
    s["m_scale"], s["v_scale"] = _scale_of(m), _scale_of(root)
    s["m"] = _rounded(m, s["m_scale"].unsqueeze(1), hi).flatten()
    codes = _rounded(root, s["v_scale"].unsqueeze(1), lo).float()
    s["v"] = torch.where((root > 0) & (codes == 0), 2.0 ** -9, codes).to(torch.float8_e4m3fn).flatten()   # a root that is not zero stays so
    return s["flat"], s["m"], s["v"], s["m_scale"], s["v_scale"]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from stag_amd import train
        if op == "scores":
            return train.row_scores(s["bits"], s["table"], s["bias"], scale=s["scale"], rows=s["rows"])
        if op == "grad":
            return train.row_scores_grad(s["bits"], s["grad"], s["n_features"], scale=s["scale"], rows=s["rows"])
        if op == "loss":
            return train.sibling_loss(s["scores"], s["label"], siblings=s["siblings"], weight=s["weight"], scale=s["scale"], grad_dtype=s["kind"])
        opt = s["opt"]
        opt.step()
        if opt.state_bits == 32:
            return s["flat"], opt.m, opt.v
        return s["flat"], opt.m, opt.v, opt.m_scale, opt.v_scale
    return {"scores": _plain_scores, "grad": _plain_grad, "loss": _plain_loss, "adamw": _plain_adamw}[op](s)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    size = DTYPES[case.get("type", "f32")].itemsize
    if op in ("scores", "grad"):
        m, k, f = case["m"], case["k"], 5 * case["ncol"]
        rows = 4 * m * _words(f) + (4 * m if case["indexed"] else 0)
        looked_up = min(f, m * case["ncol"])                                # a few rows reach a part of the table
        moved = looked_up * k * size + 4 * k + 4 * m * k if op == "scores" else m * k * size + 4 * f * k + 4 * k
        return {"bytes": rows + moved, "flops": m * case["ncol"] * k}       # one addition for each token of a row and classifier
    if op == "loss":
        m, k = case["m"], case["k"]
        read = 4 * m * k if not case["siblings"] else 4 * m * min(k, 4)     # about four siblings to a place
        return {"bytes": read + m * k * size + 4 * k + (16 if case["siblings"] else 8) * m, "flops": 12 * read // 4}
    n = sum(math.prod(shape) for shape in _shapes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": int(n * (3 * size + state)), "flops": 20 * n}


# ----------------------------------------------------------------------------------------------------------------- exact
def _exact_rows(case, seed):
    s = _prepare_rows(case, seed)
    f, m = s["n_features"], case["m"]
    rows = s["rows"].long().cpu() if s["rows"] is not None else torch.arange(m)
    values = (s["table"] if case["op"] == "scores" else s["grad"]).double()
    raw = s["bits"].view(torch.uint8)      # little-endian: bit f of a row is bit f & 7 of its byte f >> 3
    out = torch.zeros((m, case["k"]) if case["op"] == "scores" else (f, case["k"]), dtype=torch.float64, device=DEV)
    bias = torch.zeros(case["k"], dtype=torch.float64, device=DEV)
    mask = torch.tensor([1, 2, 4, 8, 16, 32, 64, 128], dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (8 * raw.shape[1]))
    for a in range(0, m, step):
        here = [i for i in range(a, min(m, a + step)) if 0 <= int(rows[i]) < s["bits"].shape[0]]
        if not here:
            continue
        at = torch.tensor(here, device=DEV)
        x = torch.bitwise_and(raw[rows[here].to(DEV)].unsqueeze(2), mask).ne(0).flatten(1)[:, :f].double()
        if case["op"] == "scores":
            out[at] = s["scale"] * torch.mm(x, values) + s["bias"].double()
        else:
            out += s["scale"] * torch.mm(x.t().contiguous(), values[at])
            bias += values[at].sum(0)
    return out if case["op"] == "scores" else (out, bias)


def _exact_loss(case, seed):
    s = _prepare_loss(case, seed)
    m, k = case["m"], case["k"]
    loss = torch.zeros(k, dtype=torch.float64, device=DEV)
    grad = torch.zeros((m, k), dtype=torch.float64, device=DEV)
    for a in range(0, m, 8192):
        z = s["scores"][a:a + 8192].double()
        y = torch.zeros_like(z)
        label = s["label"][a:a + 8192].long()
        has = label >= 0
        y[has.nonzero().flatten(), label[has]] = 1.0
        w = s["weight"][a:a + 8192].double().unsqueeze(1) * s["scale"]
        if s["siblings"] is not None:
            c = torch.arange(k, device=DEV).expand_as(z)
            w = w * ((c >= s["siblings"][a:a + 8192, 0:1]) & (c < s["siblings"][a:a + 8192, 1:2])).double()
        loss += (w * (torch.logaddexp(z, torch.zeros_like(z)) - y * z)).sum(0)
        grad[a:a + 8192] = w * (torch.sigmoid(z) - y)
    return loss, grad


def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    t, lr = s["step"] + 1, s["lr"]
    wide = lambda name: s[name].to(torch.float32).double()  # noqa: E731
    m, v, g, p = wide("m"), wide("v"), wide("grad"), wide("flat")
    if case["bits"] == 8:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    d = torch.sqrt(v / (1 - BETA2 ** t)) + EPS
    decay, l1 = (s[name].double().expand(-1, BLOCK).flatten() for name in ("decay", "l1"))
    p = p - lr * decay * p - lr * (m / (1 - BETA1 ** t)) / d
    p = torch.sign(p) * torch.clamp(p.abs() - lr * l1 / d, min=0)
    return (p, m, v) if case["bits"] == 32 else (p, None, None, None, None)      # the codes go by chance


def exact(case, seed):
    return {"scores": _exact_rows, "grad": _exact_rows, "loss": _exact_loss, "adamw": _exact_adamw}[case["op"]](case, seed)
