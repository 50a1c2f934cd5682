"""The operators around a boosted model's answers, as they are measured.

A trained model hands on two things: the leaf that each row reaches in each
tree (``predict(pred_leaf=True)``), and a score for each class.  Four operators
work on them, on tensors that are on the GPU already:

  embed       rows of a table looked up by token (a leaf of a tree, a
              category's code), summed over a row's tokens and scaled
  embed_grad  its gradient for the table
  dropout     dropout whose mask follows from a seed and an element's index
  sample      a class drawn from a row of scores with temperature, top-k,
              top-p and min-p, from a given random number per row

``run`` computes them in plain torch operations, or calls the package where
``own`` is set.  ``exact`` has the same results from the definitions in f64.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}

MIX = (0xBF58476D1CE4E5B9 - (1 << 64), 0x94D049BB133111EB - (1 << 64))  # SplitMix64's two multipliers, as int64
GAMMA = 0x9E3779B97F4A7C15 - (1 << 64)                                  # and its increment


def listed():
    return [
        # one row is scored: its leaves in 100 trees of depth 6 (127 nodes each); latency
        {"name": "embed_row", "op": "embed", "dtype": "f32", "token": "i32", "n": 1, "per_row": 100, "vocab": 12700,
         "dim": 64, "scale": 0.1, "missing": 0.0},
        # a batch on 500 trees of depth 8 (511 nodes each): the widest sum of leaf vectors
        {"name": "embed_leaves", "op": "embed", "dtype": "bf16", "token": "i32", "n": 16384, "per_row": 500,
         "vocab": 255500, "dim": 32, "scale": 0.04, "missing": 0.0},
        # one categorical column with as many codes as a column can have, an odd width, some codes missing
        {"name": "embed_codes", "op": "embed", "dtype": "f32", "token": "i64", "n": 100003, "per_row": 1,
         "vocab": 65534, "dim": 201, "scale": 14.0, "missing": 0.02},
        # a small training step on 20 categorical columns of 64 codes; latency
        {"name": "grad_codes", "op": "embed_grad", "dtype": "f32", "token": "i32", "n": 512, "per_row": 20,
         "vocab": 1280, "dim": 16, "scale": 1.0, "missing": 0.02},
        # the training step on 500 trees of depth 8: many tokens, some leaves with a large share of them
        {"name": "grad_leaves", "op": "embed_grad", "dtype": "bf16", "token": "i32", "n": 16384, "per_row": 500,
         "vocab": 255500, "dim": 32, "scale": 0.04, "missing": 0.0},
        # wide vectors of one skewed column: the commonest code holds about a tenth of the tokens
        {"name": "grad_hot", "op": "embed_grad", "dtype": "bf16", "token": "i64", "n": 32768, "per_row": 1,
         "vocab": 65534, "dim": 1024, "scale": 32.0, "missing": 0.0},
        # the smallest training step's activations; latency
        {"name": "dropout_small", "op": "dropout", "dtype": "f32", "n": 128, "dim": 64, "pad": 0, "p": 0.1},
        # activations of a large batch, an odd width inside a wider buffer
        {"name": "dropout_rows", "op": "dropout", "dtype": "bf16", "n": 65536, "dim": 1999, "pad": 1, "p": 0.2},
        # one row over a large number of classes, every limit in use; latency
        {"name": "sample_row", "op": "sample", "dtype": "f32", "n": 1, "classes": 128000, "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.02, "by_row": False, "masked": 0.0},
        # the margins of a multiclass model for a million rows
        {"name": "sample_margins", "op": "sample", "dtype": "f32", "n": 1000000, "classes": 7, "temperature": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "by_row": False, "masked": 0.0},
        # a batch over a thousand classes
        {"name": "sample_batch", "op": "sample", "dtype": "f16", "n": 2048, "classes": 1000, "temperature": 0.7,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "by_row": False, "masked": 0.0},
        # many rows over a large odd number of classes, each with its own limits, some classes ruled out
        {"name": "sample_wide", "op": "sample", "dtype": "bf16", "n": 256, "classes": 131071, "temperature": 0.9,
         "top_k": 200, "top_p": 0.95, "min_p": 0.0, "by_row": True, "masked": 0.1},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "dropout", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "dropout":
        dim = _spread(rng, 1, 8192)
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1, max(1, min(65536, 67108864 // dim))), "dim": dim,
                "pad": rng.choice([0, 0, 1, 8, 13]), "p": rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9])}
    if op == "sample":
        classes = _spread(rng, 2, 131072)
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1, max(1, min(1000000, 16777216 // classes))),
                "classes": classes, "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                "top_k": rng.choice([0, 0, 1, 5, 50, 1000]), "top_p": rng.choice([1.0, 1.0, 0.99, 0.9, 0.5]),
                "min_p": rng.choice([0.0, 0.0, 0.02, 0.2]), "by_row": rng.random() < 0.3,
                "masked": rng.choice([0.0, 0.0, 0.1, 0.9])}
    per_row = rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 64, 500)])
    dim = _spread(rng, 1, 1024) if per_row == 1 else _spread(rng, 4, 128)
    most = max(1, min(100000, 134217728 // (per_row * dim)))
    return {"op": op, "dtype": dtype, "token": rng.choice(["i32", "i64"]), "n": _spread(rng, 1, most),
            "per_row": per_row, "vocab": _spread(rng, per_row, 65534 if per_row == 1 else 511 * per_row), "dim": dim,
            "scale": rng.choice([1.0, 0.05, 8.0]), "missing": rng.choice([0.0, 0.02, 0.3])}


def _tokens(case, gen):
    """Tokens as a model gives them: column j has a range of its own (tree j's
    nodes, column j's codes), low ones of a range commoner than high ones."""
    n, k, vocab = case["n"], case["per_row"], case["vocab"]
    span = vocab // k
    u = torch.rand((n, k), generator=gen, device="cuda", dtype=torch.float64)
    if k == 1:  # one skewed column: density falls as 1 / code
        tok = (span ** u - 1).long()
    else:  # leaves of a tree: the sizes of a range's leaves differ by a factor of ten or so
        tok = (span * (1 - u.square()) * 0.999999).long()
    tok = tok.clamp_(0, span - 1) + span * torch.arange(k, device="cuda")
    if case["missing"]:
        tok[torch.rand((n, k), generator=gen, device="cuda") < case["missing"]] = -1
    tok = tok.to(torch.int32 if case["token"] == "i32" else torch.int64)
    return tok if k > 1 else tok[:, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "embed":
        state["tokens"] = _tokens(case, gen)
        state["table"] = torch.randn((case["vocab"], case["dim"]), generator=gen, device="cuda").to(dtype)
    elif case["op"] == "embed_grad":
        state["tokens"] = _tokens(case, gen)
        state["grad"] = torch.randn((case["n"], case["dim"]), generator=gen, device="cuda").to(dtype)
    elif case["op"] == "dropout":
        wide = torch.randn((case["n"], case["dim"] + case["pad"]), generator=gen, device="cuda").to(dtype)
        state["x"] = wide[:, :case["dim"]]
        state["seed"] = int(torch.randint(0, 1 << 62, (1,), generator=gen, device="cuda").item())
        state["offset"] = 1000 * (int(seed) % 1000)
    else:
        n, k = case["n"], case["classes"]
        scores = 2.0 * torch.randn((n, k), generator=gen, device="cuda")
        if case["masked"]:
            scores[torch.rand((n, k), generator=gen, device="cuda") < case["masked"]] = -math.inf
            scores[n // 2] = -math.inf  # a row that is ruled out whole
        state["logits"] = scores.to(dtype)
        state["u"] = torch.rand(n, generator=gen, device="cuda")
        for name in ("temperature", "top_k", "top_p", "min_p"):
            state[name] = case[name]
        if case["by_row"]:  # each row's own limits: the case's, looser or tighter
            loose = torch.randint(0, 4, (n,), generator=gen, device="cuda")
            state["temperature"] = case["temperature"] * (0.5 + 0.25 * loose.float())
            state["top_k"] = (case["top_k"] * loose).to(torch.int32)
            state["top_p"] = (case["top_p"] + 0.05 * (loose == 2)).float()
            state["min_p"] = case["min_p"] * (loose > 0).float()
    return state


def _own_run(state):
    from ferrisboost_b200 import ops
    case = state["case"]
    if case["op"] == "embed":
        return ops.embed(state["table"], state["tokens"], scale=case["scale"])
    if case["op"] == "embed_grad":
        return ops.embed_grad(state["grad"], state["tokens"], case["vocab"], scale=case["scale"])
    if case["op"] == "dropout":
        return ops.dropout(state["x"], case["p"], state["seed"], state["offset"])
    classes, probs = ops.sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                top_p=state["top_p"], min_p=state["min_p"])
    return {"classes": classes, "probs": probs}


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["op"] == "embed":
        return _plain_embed(state["table"], state["tokens"], case)
    if case["op"] == "embed_grad":
        return _plain_embed_grad(state["grad"], state["tokens"], case)
    if case["op"] == "dropout":
        return _plain_dropout(state["x"], case["p"], state["seed"], state["offset"])
    return _plain_sample(state)


def _plain_embed(table, tokens, case):
    # out[r] = scale * sum over the row's tokens t in [0, vocab) of table[t]
    tok = tokens.reshape(case["n"], -1).long()
    found = (tok >= 0) & (tok < case["vocab"])
    rows = table[tok.clamp(0, case["vocab"] - 1)].float() * found[:, :, None]
    return (rows.sum(1) * case["scale"]).to(table.dtype)


def _plain_embed_grad(grad, tokens, case):
    # d_table[t] = scale * sum over the places (r, j) that hold token t of grad[r]
    tok = tokens.reshape(-1).long()
    found = (tok >= 0) & (tok < case["vocab"])
    row = torch.arange(case["n"], device="cuda").repeat_interleave(case["per_row"])
    d_table = torch.zeros((case["vocab"], case["dim"]), device="cuda")
    d_table.index_add_(0, tok.clamp(0, case["vocab"] - 1), grad[row].float() * found[:, None])
    return (d_table * case["scale"]).to(grad.dtype)


def _mix(z):
    z = (z ^ ((z >> 30) & 0x3FFFFFFFF)) * MIX[0]
    z = (z ^ ((z >> 27) & 0x1FFFFFFFFF)) * MIX[1]
    return z ^ ((z >> 31) & 0x1FFFFFFFF)


def _plain_dropout(x, p, seed, offset):
    # element e = offset + its index in x has the 32 random bits of half e % 2 of word e // 2 of a
    # SplitMix64 sequence that starts at the mixed seed; it is kept where they are at least p * 2^32
    key = _mix(torch.full((1,), seed, device="cuda", dtype=torch.int64))
    e = offset + torch.arange(x.numel(), device="cuda").reshape(x.shape)
    bits = (_mix(key + ((e >> 1) + 1) * GAMMA) >> (32 * (e & 1))) & 0xFFFFFFFF
    kept = bits >= int(math.ceil(p * 4294967296.0))
    scale = torch.tensor(1.0 / (1.0 - p), device="cuda", dtype=torch.float32)
    return torch.where(kept, x.float() * scale, 0.0).to(x.dtype)


def _column(value, n, dtype):
    if isinstance(value, torch.Tensor):
        return value.to(dtype)[:, None]
    return torch.full((n, 1), value, device="cuda", dtype=dtype)


def _plain_sample(state):
    n, k = state["logits"].shape
    x = state["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    temperature = _column(state["temperature"], n, torch.float32)
    top_k = _column(state["top_k"], n, torch.int64)
    top_p = _column(state["top_p"], n, torch.float32)
    min_p = _column(state["min_p"], n, torch.float32)
    # weights relative to the row's maximum, in units of 2^-40: their sums are whole numbers, so they do not
    # depend on an order; temperature 0 leaves the first maximum only
    top = x.amax(1, keepdim=True)
    e = torch.where(x == top, 1.0, ((x - top) * (1.0 / temperature)).exp())
    e = torch.where(x == -math.inf, 0.0, e)
    w = (e * 2.0 ** 40).long()
    order = x.sort(dim=1, descending=True, stable=True).indices  # equal scores: lowest class first
    w, e = w.gather(1, order), e.gather(1, order)
    rank = torch.arange(k, device="cuda")[None, :]
    limit = torch.where(temperature == 0.0, 1, torch.where(top_k > 0, top_k, k))
    w = torch.where(rank < limit, w, 0)
    enough = (top_p.double() * w.sum(1, keepdim=True).double()).ceil().long().clamp(min=1)
    before = w.cumsum(1) - w
    w = torch.where((before < enough) | (top_p >= 1.0), w, 0)
    w = torch.where(e >= min_p, w, 0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    upto = kept.cumsum(1)
    total = upto[:, -1:]
    place = torch.minimum((state["u"].double()[:, None] * total.double()).long(), total - 1)
    drawn = (upto <= place).sum(1, keepdim=True).clamp(max=k - 1)
    probs = torch.where(total > 0, kept.gather(1, drawn).double() / total.double(), 0.0).float()
    classes = torch.where(total > 0, drawn, -1).to(torch.int32)
    return {"classes": classes[:, 0], "probs": probs[:, 0]}


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] in ("embed", "embed_grad"):
        places = case["n"] * case["per_row"]
        table = case["vocab"] if case["op"] == "embed_grad" else min(case["vocab"], places)
        return {"bytes": places * SIZES[case["token"]] + (case["n"] + table) * case["dim"] * size,
                "flops": places * case["dim"] + (case["n"] if case["op"] == "embed" else table) * case["dim"]}
    if case["op"] == "dropout":
        return {"bytes": 2 * case["n"] * case["dim"] * size, "flops": case["n"] * case["dim"]}
    limits = 16 if case["by_row"] else 0
    return {"bytes": case["n"] * (case["classes"] * size + 4 + 8 + limits), "flops": 4 * case["n"] * case["classes"]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embed":
        # one column of tokens after another, in f64; token -1 is the zero row at the end
        table = torch.cat([state["table"].double(), torch.zeros((1, case["dim"]), device="cuda", dtype=torch.float64)])
        tok = state["tokens"].reshape(case["n"], case["per_row"]).long()
        total = torch.zeros((case["n"], case["dim"]), device="cuda", dtype=torch.float64)
        for j in range(case["per_row"]):
            total += table[tok[:, j]]
        return total * case["scale"]
    if case["op"] == "embed_grad":
        # one column of tokens after another, each row's gradient to its token's sum; row `vocab` takes the missing
        tok = state["tokens"].reshape(case["n"], case["per_row"]).long()
        tok = torch.where(tok < 0, case["vocab"], tok)
        total = torch.zeros((case["vocab"] + 1, case["dim"]), device="cuda", dtype=torch.float64)
        for j in range(case["per_row"]):
            total.index_add_(0, tok[:, j], state["grad"].double(), alpha=case["scale"])
        return total[:-1]
    if case["op"] == "dropout":
        # the mask from whole words of the sequence, two elements each
        count, first = case["n"] * case["dim"], state["offset"] // 2
        words = torch.arange(first, (state["offset"] + count) // 2 + 1, device="cuda")
        z = torch.tensor([state["seed"]], device="cuda")
        for step in range(2):
            z = z if step == 0 else key + (words + 1) * GAMMA
            z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * MIX[0]
            z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * MIX[1]
            key = z = z ^ ((z >> 31) & ((1 << 33) - 1))
        halves = torch.stack([z & 0xFFFFFFFF, (z >> 32) & 0xFFFFFFFF], 1).reshape(-1)
        at = state["offset"] - 2 * first
        share = halves[at:at + count].reshape(case["n"], case["dim"]).double() / 2.0 ** 32
        return state["x"].double() / (1.0 - case["p"]) * (share >= case["p"])
    # sample: the limits on probabilities in f64, and the inverse of their sum over the classes, a few rows at a time
    n, k = case["n"], case["classes"]
    per = max(1, 33554432 // k)
    got = []
    for a in range(0, n, per):
        part = {m: v[a:a + per, None] if isinstance(v, torch.Tensor) else v for m, v in state.items() if m != "case"}
        x = state["logits"][a:a + per].double()
        t = part["temperature"]
        t = t.double() if isinstance(t, torch.Tensor) else torch.full((len(x), 1), float(torch.tensor(t)), device="cuda",
                                                                      dtype=torch.float64)
        x = torch.where(x == -math.inf, x, (x - x.amax(1, keepdim=True)) / t.clamp(min=1e-300))
        ps, order = torch.softmax(x, 1).nan_to_num(0.0).sort(dim=1, descending=True, stable=True)
        top_k = part["top_k"]
        top_k = top_k.long() if isinstance(top_k, torch.Tensor) else torch.full((len(x), 1), top_k, device="cuda")
        top_k = torch.where(t == 0, 1, torch.where(top_k > 0, top_k, k))
        ps = ps * (torch.arange(k, device="cuda") < top_k)
        ps = ps / ps.sum(1, keepdim=True).clamp(min=1e-300)
        top_p = part["top_p"].double() if isinstance(part["top_p"], torch.Tensor) else part["top_p"]
        min_p = part["min_p"].double() if isinstance(part["min_p"], torch.Tensor) else part["min_p"]
        below = ps.cumsum(1) - ps
        low = ps < min_p * ps[:, :1]
        cut = (below >= top_p) if isinstance(top_p, torch.Tensor) else (below >= (top_p if top_p < 1 else 2.0))
        if isinstance(top_p, torch.Tensor):
            cut = cut & (top_p < 1)
        ps = torch.where(cut | low, 0.0, ps)
        p = torch.zeros_like(ps).scatter_(1, order, ps)
        upto = p.cumsum(1)
        drawn = torch.searchsorted(upto, part["u"].double() * upto[:, -1:], right=True).clamp(max=k - 1)
        got.append((p.gather(1, drawn) / upto[:, -1:].clamp(min=1e-300))[:, 0])
    return {"classes": None, "probs": torch.cat(got)}
