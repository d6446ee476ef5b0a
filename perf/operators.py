"""Performance cases of the row operators that learn: embedding rows looked up by id with their gradient, and rows sorted
by expert (or node type), handed out and brought back with weights, with their gradients.

Every case makes its inputs from a seed.  `run` is one pass: in plain torch operations where `own` is false, through the
public entry points (`graph_sampling_b200.gs.nn` and `graph_sampling_b200.ops`) where it is true.
"""
import math
import random

import torch

own = False

SHAPE_SEED = 20_241  # of what has to be the same for every seed: how often each id occurs, which slots are padding
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # serving, one step: the next token of 64 sequences (or 64 seed nodes), rows scaled by the root of their width
        {"name": "lookup_step", "op": "lookup", "rows": 100_000, "width": 1024, "ids": 64, "steps": 0, "dtype": "bfloat16",
         "skew": 1.05, "padding": "none", "scale": 32.0},
        # the feature rows of a frontier in bf16; 602 values a row, so rows start on 4-byte boundaries only
        {"name": "lookup_frontier", "op": "lookup", "rows": 2_450_000, "width": 602, "ids": 1_000_000, "steps": 0,
         "dtype": "bfloat16", "skew": 0.75, "padding": "none", "scale": 1.0},
        # a training minibatch of 1 024 nodes on a small graph: lookup, then the gradient of the whole table
        {"name": "train_minibatch", "op": "train", "rows": 100_000, "width": 256, "ids": 1024, "steps": 0, "dtype": "float32",
         "skew": 0.75, "padding": "none", "scale": 1.0},
        # token embeddings of a language model's step: frequent tokens, scaled rows, id 0 is padding
        {"name": "train_tokens", "op": "train", "rows": 65_536, "width": 1024, "ids": 16_384, "steps": 0, "dtype": "bfloat16",
         "skew": 1.05, "padding": "zero", "scale": 32.0},
        # node embeddings learned from walks of 81 positions; walks that ended early are filled with -1
        {"name": "train_walks", "op": "train", "rows": 2_450_000, "width": 128, "ids": 4_050_000, "steps": 81,
         "dtype": "float32", "skew": 0.75, "padding": "minus", "scale": 1.0},
        # gradient rows of a sampled frontier for an optimizer that touches only them; 100 floats a row
        {"name": "rows_frontier", "op": "rows", "rows": 2_450_000, "width": 100, "ids": 20_011, "steps": 0, "dtype": "float32",
         "skew": 0.75, "padding": "none", "scale": 1.0},
        # the same for a table of which a dense gradient would not be affordable, positions of walks with their ends missing
        {"name": "rows_large_table", "op": "rows", "rows": 111_000_000, "width": 128, "ids": 1_000_003, "steps": 0,
         "dtype": "bfloat16", "skew": 0.75, "padding": "minus", "scale": 1.0},
        # serving, one step: 16 tokens to two of 8 experts each
        {"name": "dispatch_step", "op": "dispatch", "tokens": 16, "per_token": 2, "experts": 8, "width": 1024,
         "dtype": "bfloat16", "skew": 0.5, "dropped": 0.0},
        # a prefill batch: 64 experts, four per token
        {"name": "dispatch_batch", "op": "dispatch", "tokens": 16_384, "per_token": 4, "experts": 64, "width": 2048,
         "dtype": "bfloat16", "skew": 0.5, "dropped": 0.0},
        # serving, one step: the experts' answers brought back for 33 tokens
        {"name": "combine_step", "op": "combine", "tokens": 33, "per_token": 2, "experts": 8, "width": 1024,
         "dtype": "bfloat16", "skew": 0.5, "dropped": 0.0, "weights": "float32"},
        # a training step over a padded batch: an odd number of tokens, eight experts each, all gradients
        {"name": "experts_train", "op": "experts", "tokens": 8191, "per_token": 8, "experts": 64, "width": 1024,
         "dtype": "bfloat16", "skew": 0.5, "dropped": 0.1, "weights": "float32"},
        # nodes of a heterogeneous frontier sorted by type, projected type by type, and back: one type per node, no weights
        {"name": "types_train", "op": "experts", "tokens": 500_000, "per_token": 1, "experts": 4, "width": 256,
         "dtype": "float32", "skew": 1.0, "dropped": 0.0, "weights": "none"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "train", "train", "rows", "dispatch", "combine", "experts", "experts"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    case = {"op": op, "dtype": dtype}
    width = rng.choice([_log(rng, 1, 2048), 64, 100, 128, 256, 512, 602, 1024, 2048])
    size = 4 if dtype == "float32" else 2
    if op in ("lookup", "train", "rows"):
        most_rows = min(111_000_000 if op == "rows" else 2_450_000, (1 << 40 if op == "rows" else 1_000_000_000) // (width * size))
        rows = _log(rng, 100, most_rows)
        steps = rng.choice([0, 0, 10, 81])
        ids = _log(rng, 1, max(16, min(2_000_000, 1_000_000_000 // (width * size))))
        ids = max(steps, ids // steps * steps) if steps else ids
        case.update(rows=rows, width=width, ids=ids, steps=steps, skew=rng.choice([0.0, 0.75, 1.05]),
                    padding=rng.choice(["none", "minus", "zero"]), scale=rng.choice([1.0, 0.125, math.sqrt(width)]))
    else:
        per_token = rng.choice([1, 1, 2, 2, 3, 4, 6, 8])
        experts = max(per_token, _log(rng, 2, 256))
        tokens = _log(rng, 1, max(16, min(500_000, (1 << 25) // experts, 400_000_000 // (width * size * per_token))))
        case.update(tokens=tokens, per_token=per_token, experts=experts, width=width, skew=rng.choice([0.0, 0.5, 1.0]),
                    dropped=rng.choice([0.0, 0.0, 0.1, 0.5]))
        if op != "dispatch":
            case["weights"] = rng.choice(["float32", "float32", "same", "none"])
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------------
# Outputs of another seed have the same sizes: how often each popularity rank occurs and how many slots are padding is the
# case's, while the seed decides which id a rank has, the order of the positions and all values.
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ranks(case):
    """Popularity ranks of all positions, weight ~ (rank + 2)^-skew; -1 where a position is padding."""
    g, n = _generator(SHAPE_SEED), case["rows"] - (1 if case["padding"] == "zero" else 0)
    u = torch.rand(case["ids"], generator=g, device="cuda", dtype=torch.float64)
    power = 1.0 - case["skew"]
    low, high = 2.0 ** power, (n + 2.0) ** power
    ranks = u.mul_(high - low).add_(low).pow_(1.0 / power).sub_(2.0).to(torch.int64).clamp_(0, n - 1)
    if case["padding"] != "none":
        hidden = torch.rand(case["ids"], generator=g, device="cuda") < 0.1
        hidden[0] = False
        ranks[hidden] = -1
    return ranks


def _ids(case, seed, g):
    pick, n = random.Random(seed), case["rows"] - (1 if case["padding"] == "zero" else 0)
    stride, offset = int(n * pick.uniform(0.3, 0.7)) | 1, pick.randrange(n)
    while math.gcd(stride, n) != 1:
        stride += 2
    ranks = _ranks(case)
    ranks = ranks[torch.randperm(ranks.numel(), generator=g, device="cuda")]
    ids = ranks.mul(stride).add_(offset).remainder_(n)
    if case["padding"] == "zero":
        ids = torch.where(ranks < 0, 0, ids + 1)
    elif case["padding"] == "minus":
        ids = torch.where(ranks < 0, -1, ids)
    return ids.view(-1, case["steps"]) if case["steps"] else ids


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _experts(case, g):
    """Each token's experts, distinct, favourites among them; -1 for tokens that are padding.  float32 scores of the choices."""
    T, E = case["tokens"], case["experts"]
    favour = torch.arange(E, device="cuda", dtype=torch.float32).add_(1.0).log_().mul_(-case["skew"])
    score, ids = torch.rand((T, E), generator=g, device="cuda").log_().neg_().log_().neg_().add_(favour).topk(case["per_token"], 1)
    ids = ids.contiguous()
    ids[_dropped(case)] = -1
    return ids, score


def _dropped(case):
    """The tokens that are padding: never all of them."""
    dropped = torch.rand(case["tokens"], generator=_generator(SHAPE_SEED), device="cuda") < case["dropped"]
    dropped[0] = False
    return dropped


def prepare(case, seed):
    g, dtype, op = _generator(seed), DTYPES[case["dtype"]], case["op"]
    state = {"case": case}
    if op in ("lookup", "train", "rows"):
        state["ids"] = _ids(case, seed, g)
        state["padding"] = {"none": None, "minus": -1, "zero": 0}[case["padding"]]
        if op != "rows":
            state["table"] = _normal((case["rows"], case["width"]), g, dtype).requires_grad_(op == "train")
        if op != "lookup":
            state["grad"] = _normal((*state["ids"].shape, case["width"]), g, dtype).mul_(0.0625)
        return state
    T, K, D = case["tokens"], case["per_token"], case["width"]
    state["experts"], score = _experts(case, g)
    if op != "combine":
        state["x"] = _normal((T, D), g, dtype).requires_grad_(op == "experts")
    if op != "dispatch":
        state["y"] = _normal((T * K, D), g, dtype).requires_grad_(op == "experts")
        kind = case["weights"]
        state["weights"] = None
        if kind != "none":
            state["weights"] = torch.softmax(score, 1).to(dtype if kind == "same" else torch.float32).requires_grad_(op == "experts")
    if op == "combine":
        state["place"] = _plain_order(state["experts"], case["experts"])[2]
    if op == "experts":
        state["grad_rows"] = _normal((T * K, D), g, dtype)
        state["grad_out"] = _normal((T, D), g, dtype)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------------
def _plain_lookup(table, ids, scale, padding):
    rows = table.detach()[ids.clamp(0, table.shape[0] - 1)].float() * scale
    if padding is not None:
        rows = torch.where((ids == padding)[..., None], 0.0, rows)
    return rows.to(table.dtype)


def _plain_grad(grad, ids, rows, scale, padding):
    """Sums in 64 bits: a hub or a frequent token has tens of thousands of summands."""
    ids, grad = ids.reshape(-1), grad.reshape(-1, grad.shape[-1])
    if padding is not None:
        keep = ids != padding
        ids, grad = ids[keep], grad[keep]
    total = torch.zeros((rows, grad.shape[1]), dtype=torch.float64, device=grad.device)
    return total.index_add_(0, ids, grad.double()).mul_(scale).to(grad.dtype)


def _plain_grad_rows(grad, ids, scale, padding):
    ids, grad = ids.reshape(-1), grad.reshape(-1, grad.shape[-1])
    if padding is not None:
        keep = ids != padding
        ids, grad = ids[keep], grad[keep]
    ids, order = torch.sort(ids, stable=True)
    head = torch.ones_like(ids, dtype=torch.bool)
    head[1:] = ids[1:] != ids[:-1]
    row_ids = ids[head]
    total = torch.zeros((row_ids.numel(), grad.shape[1]), dtype=torch.float64, device=grad.device)
    total.index_add_(0, torch.cumsum(head, 0) - 1, grad[order].double())
    return row_ids, total.mul_(scale).to(grad.dtype)


def _plain_order(experts, num_experts):
    """(offsets, source, place): rows of expert e are offsets[e] .. offsets[e + 1], in the order of their slots, dropped slots
    behind the last; source[row] = slot, place[slot] = row, or -1 - row for a dropped slot."""
    key = experts.reshape(-1)
    key = torch.where(key < 0, num_experts, key)
    source = torch.argsort(key, stable=True)
    place = torch.empty_like(source)
    place[source] = torch.arange(source.numel(), device=key.device)
    place = torch.where(key == num_experts, -1 - place, place).view_as(experts)
    count = (key[:, None] == torch.arange(num_experts, device=key.device)).sum(0)
    offsets = torch.zeros(num_experts + 1, dtype=torch.int64, device=key.device)
    offsets[1:] = torch.cumsum(count, 0)
    return offsets, source, place


def _plain_spread(x, place, weights=None):
    """rows[place[t, k]] = weights[t, k] * x[t]; zeros in the rows of dropped slots."""
    T, K = place.shape
    values = x.detach().float()[:, None, :].expand(T, K, -1)
    if weights is not None:
        values = values * weights.detach().float()[..., None]
    values = torch.where((place < 0)[..., None], 0.0, values)
    rows = torch.empty((T * K, x.shape[1]), dtype=x.dtype, device=x.device)
    rows[torch.where(place < 0, -1 - place, place).reshape(-1)] = values.reshape(T * K, -1).to(x.dtype)
    return rows


def _plain_brought(rows, place):
    """rows[place[t, k]] in 32 bits, zeros for dropped slots."""
    return torch.where((place < 0)[..., None], 0.0, rows.detach()[place.clamp(min=0)].float())


def _plain_combine(rows, place, weights=None):
    brought = _plain_brought(rows, place)
    if weights is not None:
        brought = brought * weights.detach().float()[..., None]
    return brought.sum(1).to(rows.dtype)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("lookup", "train"):
        out = _plain_lookup(s["table"], s["ids"], case["scale"], s["padding"])
        if op == "lookup":
            return {"out": out}
        return {"out": out, "grad": _plain_grad(s["grad"], s["ids"], case["rows"], case["scale"], s["padding"])}
    if op == "rows":
        row_ids, rows = _plain_grad_rows(s["grad"], s["ids"], case["scale"], s["padding"])
        return {"row_ids": row_ids, "rows": rows}
    if op == "combine":
        return {"out": _plain_combine(s["y"], s["place"], s["weights"])}
    offsets, source, place = _plain_order(s["experts"], case["experts"])
    out = {"offsets": offsets, "source": source, "place": place, "rows": _plain_spread(s["x"], place)}
    if op == "experts":
        w = s["weights"]
        out["out"] = _plain_combine(s["y"], place, w)
        out["grad_x"] = _plain_combine(s["grad_rows"], place)
        out["grad_y"] = _plain_spread(s["grad_out"], place, w)
        if w is not None:
            out["grad_weights"] = (s["grad_out"].float()[:, None, :] * _plain_brought(s["y"], place)).sum(2).to(w.dtype)
    return out


# ---- the framework's calls -------------------------------------------------------------------------------------------------
def _run_own(s):
    from graph_sampling_b200 import ops
    from graph_sampling_b200.gs import nn
    case = s["case"]
    op = case["op"]
    if op == "lookup":
        return {"out": ops.embedding_lookup(s["table"], s["ids"], case["scale"], s["padding"])}
    if op == "train":
        out = nn.embedding(s["table"], s["ids"], case["scale"], s["padding"])
        grad, = torch.autograd.grad(out, s["table"], s["grad"])
        return {"out": out, "grad": grad}
    if op == "rows":
        row_ids, rows = ops.embedding_grad_rows(s["grad"], s["ids"], case["rows"], case["scale"], s["padding"])
        return {"row_ids": row_ids, "rows": rows}
    if op == "combine":
        return {"out": ops.expert_combine(s["y"], s["place"], s["weights"])}
    if op == "dispatch":
        offsets, source, place = ops.expert_order(s["experts"], case["experts"])
        return {"offsets": offsets, "source": source, "place": place, "rows": ops.expert_dispatch(s["x"], place)}
    offsets, source, place = ops.expert_order(s["experts"], case["experts"])
    rows = nn.dispatch(s["x"], place)
    out = nn.combine(s["y"], place, s["weights"])
    wanted = [s["x"], s["y"]] + ([] if s["weights"] is None else [s["weights"]])
    grads = torch.autograd.grad((rows, out), wanted, (s["grad_rows"], s["grad_out"]))
    got = {"offsets": offsets, "source": source, "place": place, "rows": rows, "out": out, "grad_x": grads[0], "grad_y": grads[1]}
    if s["weights"] is not None:
        got["grad_weights"] = grads[2]
    return got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass has to read, write and compute ------------------------------------------------------------------------------
def work(case):
    size, op, D = 4 if case["dtype"] == "float32" else 2, case["op"], case["width"]
    if op in ("lookup", "train", "rows"):
        ranks = _ranks(case)
        kept = int((ranks >= 0).sum())
        distinct = int(torch.unique(ranks[ranks >= 0]).numel())
        row, n = D * size, case["ids"]
        lookup = 8 * n + distinct * row + n * row
        if op == "lookup":
            return {"bytes": lookup, "flops": n * D}
        if op == "rows":
            return {"bytes": 8 * n + kept * row + distinct * (8 + row), "flops": kept * D}
        return {"bytes": lookup + kept * row + case["rows"] * row, "flops": 2 * n * D}
    T, K = case["tokens"], case["per_token"]
    row, n = D * size, T * K
    kept = K * (T - int(_dropped(case).sum()))
    weights = {"none": 0, "same": size, "float32": 4}[case.get("weights", "none")] * n
    order = 8 * n + 8 * (case["experts"] + 1) + 16 * n
    if op == "dispatch":
        return {"bytes": order + T * row + n * row, "flops": 0}
    combine = kept * row + weights + T * row
    if op == "combine":
        return {"bytes": 8 * n + combine, "flops": 2 * kept * D}
    # dispatch, combine, and back: the gradient of x sums rows, that of y spreads and that of the weights multiplies with y
    # again (read once), the gradient of the output is read once
    back = kept * row + T * row + T * row + n * row + 2 * weights
    return {"bytes": order + T * row + n * row + combine + back, "flops": 6 * kept * D}


# ---- the operators' definition in 64 bits -------------------------------------------------------------------------------------
def _exact_sums(grad, ids, padding):
    """(distinct ids, ascending, and the sums of their gradients in 64 bits), segment by segment of the sorted ids."""
    ids, grad = ids.flatten(), grad.flatten(0, -2)
    live = torch.nonzero(ids != (-(1 << 62) if padding is None else padding)).squeeze(1)
    row_ids, count = torch.unique(ids[live], return_counts=True)
    by_id = live[torch.argsort(ids[live])]
    return row_ids, torch.segment_reduce(grad.index_select(0, by_id).double(), "sum", lengths=count, axis=0)


def exact(case, seed):
    s = prepare(case, seed)
    op, out = case["op"], {}
    if op in ("lookup", "train"):
        table, ids = s["table"].detach(), s["ids"].flatten()
        alive = torch.ones_like(ids) if s["padding"] is None else (ids - s["padding"]).ne(0).long()
        rows = table.index_select(0, ids * alive).double()
        out["out"] = rows.mul_(case["scale"]).mul_(alive[:, None]).view(*s["ids"].shape, -1)
    if op in ("train", "rows"):
        row_ids, sums = _exact_sums(s["grad"], s["ids"], s["padding"])
        sums *= case["scale"]
        if op == "rows":
            return {"row_ids": row_ids, "rows": sums}
        out["grad"] = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda").index_copy_(0, row_ids, sums)
    if op in ("lookup", "train"):
        return out
    T, K, D, E = case["tokens"], case["per_token"], case["width"], case["experts"]
    flat = s["experts"].flatten().tolist()
    lists = [[] for _ in range(E + 1)]
    for slot, e in enumerate(flat):
        lists[e].append(slot)  # -1: the last list
    source = torch.tensor([slot for some in lists for slot in some], dtype=torch.int64, device="cuda").reshape(-1)
    place = torch.empty_like(source).index_copy_(0, source, torch.arange(T * K, device="cuda"))
    ends = [0]
    for some in lists[:E]:
        ends.append(ends[-1] + len(some))
    alive = torch.tensor([1.0 if e >= 0 else 0.0 for e in flat], dtype=torch.float64, device="cuda").view(T, K)
    at, token = place.view(T, K), source.div(K, rounding_mode="floor")
    live = alive.flatten().index_select(0, source)[:, None]
    w = None if s.get("weights") is None else s["weights"].detach().double()

    def back(rows, factor):
        total = torch.zeros(T, D, dtype=torch.float64, device="cuda")
        for k in range(K):
            total += rows.detach().index_select(0, at[:, k]).double() * factor[:, k:k + 1]
        return total

    if op != "combine":
        out = {"offsets": torch.tensor(ends, dtype=torch.int64, device="cuda"), "source": source,
               "place": torch.where(alive > 0, at, ~at), "rows": s["x"].detach().index_select(0, token).double() * live}
    if op != "dispatch":
        out["out"] = back(s["y"], alive if w is None else alive * w)
    if op == "experts":
        out["grad_x"] = back(s["grad_rows"], alive)
        factor = live if w is None else live * w.flatten().index_select(0, source)[:, None]
        out["grad_y"] = s["grad_out"].index_select(0, token).double() * factor
        if w is not None:
            dots = (s["grad_out"].index_select(0, token).double() * s["y"].detach().double()).sum(1)
            out["grad_weights"] = torch.empty_like(dots).index_copy_(0, source, dots).view(T, K) * alive
    return out
