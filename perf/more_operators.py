"""Performance cases of what runs over rows sorted by expert (or node type): their matrix products with one weight matrix per
expert, with gradients; the same products in 8-bit integers with a scale per row and per output channel; and dropout whose mask
comes from a counter-based generator and is never stored.

Every case makes its inputs from a seed.  `run` is one pass: in plain torch operations where `own` is false, through the
public entry points (`graph_sampling_b200.gs.nn` and `graph_sampling_b200.ops`) where it is true.
"""
import math
import random

import torch

own = False

SHAPE_SEED = 31_415  # of what has to be the same for every seed: how many rows the experts have
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MASK32 = 0xFFFFFFFF
DROPOUT_STREAM = 6   # the generator's operator tag


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # serving, one step: 16 tokens, two of 8 experts each; bound by the experts' weights
        {"name": "product_step", "op": "product", "rows": 32, "experts": 8, "k": 1024, "n": 2048, "dtype": "bfloat16",
         "skew": 0.5, "dropped": 0.0},
        # a prefill batch: 16 384 tokens, four of 64 experts each
        {"name": "product_batch", "op": "product", "rows": 65_536, "experts": 64, "k": 2048, "n": 2048, "dtype": "bfloat16",
         "skew": 0.5, "dropped": 0.0},
        # feature rows of a heterogeneous frontier (602 values) projected type by type to 100; nothing is a multiple of 16 bytes
        {"name": "product_frontier", "op": "product", "rows": 200_003, "experts": 7, "k": 602, "n": 100, "dtype": "float16",
         "skew": 1.0, "dropped": 0.05},
        # a training minibatch of 1 024 nodes of three types, small layer in float32
        {"name": "train_minibatch", "op": "train", "rows": 1024, "experts": 3, "k": 100, "n": 47, "dtype": "float32",
         "skew": 0.5, "dropped": 0.0},
        # a training step over a padded batch: 8 191 tokens, eight of 64 experts each, all gradients
        {"name": "train_experts", "op": "train", "rows": 65_528, "experts": 64, "k": 1024, "n": 1024, "dtype": "bfloat16",
         "skew": 0.5, "dropped": 0.1},
        # nodes of a heterogeneous graph projected type by type, float32, all gradients
        {"name": "train_types", "op": "train", "rows": 500_000, "experts": 4, "k": 256, "n": 256, "dtype": "float32",
         "skew": 1.0, "dropped": 0.0},
        # serving in 8 bits, one step: 33 tokens, two of 8 experts each, rows quantized on the way
        {"name": "int8_step", "op": "int8", "rows": 66, "experts": 8, "k": 1024, "n": 2048, "dtype": "bfloat16", "skew": 0.5,
         "dropped": 0.0},
        # a prefill batch in 8 bits
        {"name": "int8_batch", "op": "int8", "rows": 65_536, "experts": 64, "k": 2048, "n": 2048, "dtype": "bfloat16",
         "skew": 0.5, "dropped": 0.0},
        # hidden rows of a small minibatch, forward and backward
        {"name": "dropout_minibatch", "op": "dropout", "rows": 1024, "k": 256, "dtype": "float32", "p": 0.5, "train": True},
        # feature rows of a large frontier, 602 values each, forward
        {"name": "dropout_frontier", "op": "dropout", "rows": 1_000_000, "k": 602, "dtype": "bfloat16", "p": 0.1, "train": False},
        # hidden rows between two products of a training step, forward and backward
        {"name": "dropout_experts", "op": "dropout", "rows": 65_528, "k": 1024, "dtype": "bfloat16", "p": 0.1, "train": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))))


def draw(rng):
    op = rng.choice(["product", "product", "train", "train", "int8", "int8", "dropout"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])

    def width():
        return rng.choice([_log(rng, 1, 2048), 64, 100, 128, 256, 512, 602, 1024, 2048])

    if op == "dropout":
        k = width()
        return {"op": op, "dtype": dtype, "k": k, "rows": _log(rng, 1, max(16, 300_000_000 // k)),
                "p": rng.choice([0.0, 0.1, 0.2, 0.5, 0.9]), "train": rng.choice([True, False])}
    k, n = width(), width()
    experts = min(_log(rng, 1, 256), max(1, 300_000_000 // (k * n)))
    rows = _log(rng, 1, max(16, min(500_000, 200_000_000 // max(k, n), 150_000_000_000 // (k * n))))
    return {"op": op, "dtype": "bfloat16" if op == "int8" and dtype == "float32" else dtype, "rows": rows, "experts": experts,
            "k": k, "n": n, "skew": rng.choice([0.0, 0.5, 1.0]), "dropped": rng.choice([0.0, 0.0, 0.1, 0.5])}


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _counts(case):
    """Rows per expert, favourites first; the rest of the rows belongs to no expert and lies behind the last one's."""
    rng, E = random.Random(SHAPE_SEED), case["experts"]
    kept = max(1, case["rows"] - int(case["rows"] * case["dropped"]))
    share = [(e + 1.0) ** -case["skew"] * rng.uniform(0.5, 1.5) for e in range(E)]
    ends, run, total = [], 0.0, sum(share)
    for s in share:
        run += s
        ends.append(int(round(kept * run / total)))
    ends[-1] = kept
    return [b - a for a, b in zip([0] + ends, ends)]


def prepare(case, seed):
    g, dtype, op = _generator(seed), DTYPES[case["dtype"]], case["op"]
    state = {"case": case}
    R, K = case["rows"], case["k"]
    if op == "dropout":
        state["seed"] = random.Random(seed).getrandbits(64)
        state["x"] = _normal((R, K), g, dtype).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = _normal((R, K), g, dtype)
        return state
    E, N = case["experts"], case["n"]
    counts = _counts(case)
    random.Random(seed).shuffle(counts)
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    state["ends"] = ends                                   # the same on the host, for the plain form
    state["offsets"] = torch.tensor(ends, dtype=torch.int64, device="cuda")
    state["x"] = _normal((R, K), g, dtype)
    state["x"][ends[-1]:] = 0                              # as dispatch leaves the rows of dropped slots
    w = torch.randn((E, K, N), generator=g, device="cuda").mul_(K ** -0.5)
    if op == "int8":                                       # quantized once, when the model is loaded
        amax = w.abs().amax(1)
        state["weight_scales"] = amax / 127.0
        q = torch.round(w / state["weight_scales"][:, None, :]).clamp_(-127, 127).to(torch.int8)
        stride = (K + 15) // 16 * 16
        held = torch.zeros((E, N, stride), dtype=torch.int8, device="cuda")
        held[:, :, :K] = q.transpose(1, 2)
        state["weight_values"] = held[:, :, :K]
        return state
    state["weights"] = w.to(dtype)
    if op == "train":
        state["x"].requires_grad_()
        state["weights"].requires_grad_()
        state["grad"] = _normal((R, N), g, dtype)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------------
def _plain_product(x, w, ends):
    """Rows ends[e] .. ends[e + 1] times w[e]; zeros in the rows of no expert."""
    out = torch.zeros((x.shape[0], w.shape[2]), dtype=x.dtype, device=x.device)
    for e in range(w.shape[0]):
        if ends[e + 1] > ends[e]:
            out[ends[e]:ends[e + 1]] = (x[ends[e]:ends[e + 1]].float() @ w[e].float()).to(x.dtype)
    return out


def _plain_grad_weights(x, grad, ends, experts):
    """Sums over all rows of an expert: in 64 bits where the result has 32."""
    wide = torch.float64 if x.dtype == torch.float32 else torch.float32
    out = torch.zeros((experts, x.shape[1], grad.shape[1]), dtype=x.dtype, device=x.device)
    for e in range(experts):
        if ends[e + 1] > ends[e]:
            out[e] = (x[ends[e]:ends[e + 1]].to(wide).t() @ grad[ends[e]:ends[e + 1]].to(wide)).to(x.dtype)
    return out


def _plain_int8(x, values, scales, ends):
    """Rows in 8 bits with a scale each, max / 127; products of whole numbers (exact in 64-bit floats), scaled back."""
    x = x.float()
    top = x.abs().amax(1)
    row_scale = top / torch.full_like(top, 127.0)         # a quotient: division by a number multiplies with its reciprocal
    q = torch.round(x / row_scale[:, None]).clamp(-127, 127)
    q = torch.where(row_scale[:, None] == 0, 0.0, q).double()
    out = torch.zeros((x.shape[0], values.shape[1]), device=x.device)
    for e in range(values.shape[0]):
        if ends[e + 1] > ends[e]:
            total = q[ends[e]:ends[e + 1]] @ values[e].double().t()
            out[ends[e]:ends[e + 1]] = total.float() * row_scale[ends[e]:ends[e + 1], None] * scales[e][None, :]
    return out


def _plain_words(seed, blocks):
    """Philox4x32-10 of counters (b, b >> 32, 0, tag), 0 <= b < blocks: four 32-bit words each."""
    c = [torch.arange(blocks, dtype=torch.int64, device="cuda"), None, None, None]
    c[1] = c[0] >> 32
    c[0] = c[0] & MASK32
    c[2] = torch.zeros_like(c[0])
    c[3] = torch.full_like(c[0], DROPOUT_STREAM)
    k0, k1 = seed & MASK32, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57         # modulo 2^64: the bits of both halves are right
        c = [((p1 >> 32) & MASK32) ^ c[1] ^ k0, p1 & MASK32, ((p0 >> 32) & MASK32) ^ c[3] ^ k1, p0 & MASK32]
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack(c, 1)


def _plain_kept(seed, count, p):
    """(which of `count` values stay, what they are multiplied with): value i belongs to the 16 bits i % 8 of block i / 8 and is
    dropped where they are below p * 65 536, rounded."""
    limit = int(math.floor(p * 65536.0 + 0.5))
    words = _plain_words(seed, (count + 7) // 8)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:count]
    return halves >= limit, 65536.0 / (65536 - limit) if limit < 65536 else 0.0


def _run_plain(s):
    case = s["case"]
    if case["op"] == "dropout":
        x = s["x"].detach()
        kept, scale = _plain_kept(s["seed"], x.numel(), case["p"])
        kept = kept.view_as(x)
        out = {"out": torch.where(kept, x.float() * scale, 0.0).to(x.dtype)}
        if case["train"]:
            out["grad"] = torch.where(kept, s["grad"].float() * scale, 0.0).to(x.dtype)
        return out
    if case["op"] == "int8":
        return {"out": _plain_int8(s["x"], s["weight_values"], s["weight_scales"], s["ends"]).to(s["x"].dtype)}
    x, w = s["x"].detach(), s["weights"].detach()
    out = {"out": _plain_product(x, w, s["ends"])}
    if case["op"] == "train":
        out["grad_rows"] = _plain_product(s["grad"], w.transpose(1, 2), s["ends"])
        out["grad_weights"] = _plain_grad_weights(x, s["grad"], s["ends"], case["experts"])
    return out


# ---- the framework's calls -------------------------------------------------------------------------------------------------
def _run_own(s):
    from graph_sampling_b200 import ops
    from graph_sampling_b200.gs import nn
    case = s["case"]
    op = case["op"]
    if op == "dropout":
        if not case["train"]:
            return {"out": ops.dropout(s["x"], case["p"], s["seed"])}
        out = nn.dropout(s["x"], case["p"], s["seed"])
        grad, = torch.autograd.grad(out, s["x"], s["grad"])
        return {"out": out, "grad": grad}
    if op == "int8":
        values, scales = ops.quantize_rows(s["x"])
        return {"out": ops.expert_product_int8(values, scales, s["weight_values"], s["weight_scales"], s["offsets"], s["x"].dtype)}
    if op == "product":
        return {"out": ops.expert_product(s["x"], s["weights"], s["offsets"])}
    out = nn.product(s["x"], s["weights"], s["offsets"])
    grad_rows, grad_weights = torch.autograd.grad(out, (s["x"], s["weights"]), s["grad"])
    return {"out": out, "grad_rows": grad_rows, "grad_weights": grad_weights}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass has to read, write and compute ------------------------------------------------------------------------------
def work(case):
    size, R, K = 4 if case["dtype"] == "float32" else 2, case["rows"], case["k"]
    if case["op"] == "dropout":
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * R * K * size, "flops": passes * R * K}
    E, N = case["experts"], case["n"]
    counts = _counts(case)
    kept, used = sum(counts), sum(c > 0 for c in counts)
    product = 2 * kept * K * N
    if case["op"] == "int8":
        return {"bytes": 8 * (E + 1) + kept * K * size + used * (K * N + 4 * N) + R * N * size, "flops": product}
    once = 8 * (E + 1) + kept * K * size + used * K * N * size + R * N * size
    if case["op"] == "product":
        return {"bytes": once, "flops": product}
    return {"bytes": once + kept * N * size + R * K * size + E * K * N * size, "flops": 3 * product}


# ---- the operators' definition in 64 bits -------------------------------------------------------------------------------------
def _exact_bits(seed, count):
    """The generator's 16 bits of every value, with products of 32-bit numbers put together from 16-bit halves."""
    def times(a, m):
        low, high = a & 0xFFFF, a >> 16
        ll, lh, hl, hh = low * (m & 0xFFFF), low * (m >> 16), high * (m & 0xFFFF), high * (m >> 16)
        middle = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
        return hh + (lh >> 16) + (hl >> 16) + (middle >> 16), (middle & 0xFFFF) << 16 | ll & 0xFFFF

    parts = []
    blocks = (count + 7) // 8
    for first in range(0, blocks, 1 << 24):
        item = torch.arange(first, min(blocks, first + (1 << 24)), device="cuda")
        a, b = item.remainder(1 << 32), item.div(1 << 32, rounding_mode="floor")
        c, d = torch.zeros_like(a), torch.zeros_like(a) + DROPOUT_STREAM
        for r in range(10):
            key0 = (seed % (1 << 32) + r * 0x9E3779B9) % (1 << 32)
            key1 = (seed // (1 << 32) + r * 0xBB67AE85) % (1 << 32)
            (high_a, low_a), (high_c, low_c) = times(a, 0xD2511F53), times(c, 0xCD9E8D57)
            a, b, c, d = high_c ^ b ^ key0, low_c, high_a ^ d ^ key1, low_a
        eight = torch.empty((item.numel(), 8), dtype=torch.int32, device="cuda")
        for j, word in enumerate((a, b, c, d)):
            eight[:, 2 * j] = word % 65536
            eight[:, 2 * j + 1] = word // 65536
        parts.append(eight.flatten())
    return torch.cat(parts)[:count]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["op"] == "dropout":
        dropped = round(case["p"] * 65536)
        factor = (_exact_bits(s["seed"], x.numel()) >= dropped).double().view_as(x)
        if dropped < 65536:
            factor *= 65536 / (65536 - dropped)
        out = {"out": x.double() * factor}
        if case["train"]:
            out["grad"] = s["grad"].double() * factor
        return out
    ends, E = s["ends"], case["experts"]
    sizes = [ends[e + 1] - ends[e] for e in range(E)] + [case["rows"] - ends[-1]]
    rows_of = torch.split(x.double(), sizes)[:E]
    rest = sizes[-1]
    if case["op"] == "int8":
        scale = x.float().abs().max(dim=1).values.double().div(127).float()
        parts = []
        for e in range(E):
            of_rows = scale[ends[e]:ends[e + 1], None].double()
            # the quotient is a 32-bit number, as the definition has it
            q = torch.nan_to_num((rows_of[e] / of_rows).float().double().round().clamp(-127, 127), nan=0.0)
            weights = s["weight_values"][e].double() * s["weight_scales"][e].double()[:, None]
            parts.append(torch.einsum("rk,nk->rn", q * of_rows, weights))
        parts.append(torch.zeros((rest, case["n"]), dtype=torch.float64, device="cuda"))
        return {"out": torch.cat(parts)}
    w = s["weights"].detach().double()
    zeros = [torch.zeros((rest, case["n"]), dtype=torch.float64, device="cuda")]
    out = {"out": torch.cat([torch.einsum("rk,kn->rn", r, w[e]) for e, r in enumerate(rows_of)] + zeros)}
    if case["op"] == "train":
        grads = torch.split(s["grad"].double(), sizes)[:E]
        zeros = [torch.zeros((rest, case["k"]), dtype=torch.float64, device="cuda")]
        out["grad_rows"] = torch.cat([torch.einsum("rn,kn->rk", g, w[e]) for e, g in enumerate(grads)] + zeros)
        out["grad_weights"] = torch.stack([torch.einsum("rk,rn->kn", r, g) for r, g in zip(rows_of, grads)])
    return out
