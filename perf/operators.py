"""Performance cases of the dense operators: the products that serve a layer's weights in 8 bits, and the optimiser's step
that trains them.

  * `linear8`: tokens and weights are 8-bit codes with a scale for each row, `int8_linear`;
  * `serve`: tokens are floating point and are coded within the call, `quantized_linear`;
  * `ortho`: an update (or a batch of them) is orthogonalised by Newton-Schulz products, `orthogonalize`;
  * `muon`: the optimiser's step of several weights of one shape, momentum and weight update included, `muon_step`.

`listed()` names twelve cases, `draw()` gives others of the same ranges.  With `own` false `run` computes them from
elementary torch operations in float32, with `own` true it calls the library.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_STEPS = 5


# ---- the cases ------------------------------------------------------------------------------------
def listed():
    return [
        # the dense part of a layer on a minibatch of 1024 seeds, inputs coded already: a call whose launch counts
        {"name": "linear8_minibatch", "kind": "linear8", "rows": 1024, "cols": 128, "outs": 256, "dtype": "float32",
         "bias": True, "relu": True},
        # a block of a graph with features of an odd width, from the table's codes
        {"name": "linear8_602", "kind": "linear8", "rows": 60001, "cols": 602, "outs": 128, "dtype": "float32",
         "bias": True, "relu": False},
        # the largest: a long batch through a wide square layer
        {"name": "linear8_large", "kind": "linear8", "rows": 16384, "cols": 8192, "outs": 8192, "dtype": "bfloat16",
         "bias": False, "relu": False},
        # one token: the weights are read once, and that is the time
        {"name": "serve_token", "kind": "serve", "rows": 1, "cols": 4096, "outs": 4096, "dtype": "bfloat16",
         "bias": True, "relu": False},
        # a few dozen tokens of different requests at a wide output
        {"name": "serve_33", "kind": "serve", "rows": 33, "cols": 4096, "outs": 16384, "dtype": "bfloat16",
         "bias": False, "relu": False},
        # a chunk of tokens, no whole number of tiles
        {"name": "serve_chunk", "kind": "serve", "rows": 4099, "cols": 4096, "outs": 4096, "dtype": "float16",
         "bias": True, "relu": True},
        # inference over all destination rows of a large block of a graph: few columns, much output
        {"name": "serve_block", "kind": "serve", "rows": 250000, "cols": 100, "outs": 128, "dtype": "float32",
         "bias": True, "relu": True},
        # a batch of small squares, a matrix per head or expert
        {"name": "ortho_batch", "kind": "ortho", "count": 48, "rows": 128, "cols": 128, "dtype": "bfloat16"},
        # a wide layer's update, rows and columns no multiples of anything
        {"name": "ortho_odd", "kind": "ortho", "count": 1, "rows": 1000, "cols": 2051, "dtype": "float32"},
        # the largest update, a square one
        {"name": "ortho_large", "kind": "ortho", "count": 1, "rows": 4096, "cols": 4096, "dtype": "bfloat16"},
        # the two weights of a GraphSAGE layer: a step that launches and latency bound
        {"name": "muon_layer", "kind": "muon", "count": 2, "rows": 256, "cols": 128, "dtype": "float32", "nesterov": True},
        # tall weights of an ordinary size, four layers together
        {"name": "muon_tall", "kind": "muon", "count": 4, "rows": 2048, "cols": 512, "dtype": "bfloat16", "nesterov": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over its logarithm, every other one a whole number of tiles."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 else max(lo, min(hi, (v + 63) // 64 * 64))


def draw(rng):
    kind = rng.choice(["linear8", "serve", "serve", "ortho", "muon"])
    case = {"kind": kind}
    if kind in ("linear8", "serve"):
        cols, outs = _size(rng, 64, 8192), _size(rng, 32, 16384)
        # from single tokens to long batches, held to 2^28 outputs and inputs and the largest case's products
        most = min(300000, (1 << 28) // max(cols, outs), (1 << 40) // (cols * outs))
        rows = _log(rng, 1, most) if rng.random() < 0.7 else _log(rng, 1, 64)
        case.update(rows=rows, cols=cols, outs=outs, dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]),
                    bias=rng.random() < 0.5, relu=rng.random() < 0.3)
    else:
        rows, cols = _size(rng, 32, 4096), _size(rng, 32, 4096)
        least = min(rows, cols)
        # as many as make half of the largest case's products at most, up to 64 (32 where a step returns two of each)
        most = max(1, min(64 if kind == "ortho" else 32, (1 << 37) // (rows * cols * least)))
        case.update(count=_log(rng, 1, most), rows=rows, cols=cols, dtype=rng.choice(["float32", "bfloat16"]))
        if kind == "muon":
            case.update(nesterov=rng.random() < 0.7)
    return case


# ---- what a caller has in hand ----------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(case, g):
    """Activations: columns of different sizes, a few of them far larger than the others, rows of different lengths."""
    column = torch.exp(0.5 * torch.randn((case["cols"],), generator=g, device="cuda"))
    column[torch.randint(0, case["cols"], (max(1, case["cols"] // 200),), generator=g, device="cuda")] *= 8
    length = torch.exp(0.3 * torch.randn((case["rows"], 1), generator=g, device="cuda"))
    return torch.randn((case["rows"], case["cols"]), generator=g, device="cuda").mul_(length).mul_(column)


def _codes(x):
    """Codes and scales of the rows of float32 x; rows of codes start at multiples of 16 bytes, as a table keeps them."""
    scales = torch.clamp(x.abs().amax(dim=1), min=1e-30) * (1 / 127)
    room = torch.zeros((x.shape[0], (x.shape[1] + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    codes = room[:, :x.shape[1]]
    codes.copy_(torch.clamp(torch.round(x * scales.reciprocal()[:, None]), -127, 127))
    return codes, scales


def _updates(case, g, dtype):
    """Gradients: a few strong directions whose sizes fall off, over noise."""
    n, rows, cols = case["count"], case["rows"], case["cols"]
    rank = max(2, min(rows, cols) // 8)
    fall = torch.logspace(0, -1.5, rank, device="cuda")
    left = torch.randn((n, rows, rank), generator=g, device="cuda") * fall
    right = torch.randn((n, rank, cols), generator=g, device="cuda")
    return ((left @ right).mul_(1e-3).add_(torch.randn((n, rows, cols), generator=g, device="cuda"), alpha=3e-4)).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] in ("linear8", "serve"):
        weight = torch.randn((case["outs"], case["cols"]), generator=g, device="cuda") / math.sqrt(case["cols"])
        state["weight_codes"], state["weight_scales"] = _codes(weight)
        state["bias"] = torch.randn((case["outs"],), generator=g, device="cuda") if case["bias"] else None
        tokens = _tokens(case, g)
        if case["kind"] == "linear8":
            state["codes"], state["scales"] = _codes(tokens)
        else:
            state["x"] = tokens.to(dtype)
        state["dtype"] = dtype
    elif case["kind"] == "ortho":
        updates = _updates(case, g, dtype)
        state["update"] = updates if case["count"] > 1 else updates[0]
    else:
        shape = (case["rows"], case["cols"])
        grads = _updates(case, g, dtype)
        state["grads"] = [grads[i].clone() for i in range(case["count"])]
        state["momenta"] = [torch.randn(shape, generator=g, device="cuda") * 3e-4 for _ in range(case["count"])]
        state["weights"] = [(torch.randn(shape, generator=g, device="cuda") / math.sqrt(case["cols"])).to(dtype)
                            for _ in range(case["count"])]
    return state


# ---- one pass ---------------------------------------------------------------------------------------
_STEP_SIZE, _DECAY, _MOMENTUM = 0.02, 0.0002, 0.95


def _plain_product(codes, scales, s):
    out = (codes @ s["weight_codes"].float().t()) * (scales[:, None] * s["weight_scales"])
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["relu"]:
        out = torch.clamp(out, min=0)
    return out.to(s["dtype"])


def _plain_orthogonal(u):
    """Newton-Schulz iteration of float32 matrices [..., rows, cols]."""
    a, b, c = _COEFFICIENTS
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(_STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain(s):
    if s["kind"] == "linear8":
        return _plain_product(s["codes"].float(), s["scales"], s)
    if s["kind"] == "serve":
        x = s["x"].float()
        scales = torch.clamp(x.abs().amax(dim=1), min=1e-30) * (1 / 127)
        return _plain_product(torch.clamp(torch.round(x * scales.reciprocal()[:, None]), -127, 127), scales, s)
    if s["kind"] == "ortho":
        return _plain_orthogonal(s["update"].float()).to(s["update"].dtype)
    grad, held = torch.stack(s["grads"]).float(), torch.stack(s["momenta"])
    held = _MOMENTUM * held + (1 - _MOMENTUM) * grad
    update = _MOMENTUM * held + (1 - _MOMENTUM) * grad if s["nesterov"] else held
    weight = (1 - _DECAY) * torch.stack(s["weights"]).float() - _STEP_SIZE * _plain_orthogonal(update)
    torch._foreach_copy_(s["momenta"], list(held.unbind()))
    torch._foreach_copy_(s["weights"], list(weight.to(s["weights"][0].dtype).unbind()))
    return {"weights": s["weights"], "momenta": s["momenta"]}


def run(state):
    s = state
    if not own:
        return _plain(s)
    import f2cgt_amd
    lib = f2cgt_amd.load()
    if s["kind"] == "linear8":
        return lib.int8_linear(s["codes"], s["scales"], s["weight_codes"], s["weight_scales"], s["bias"], s["relu"], s["dtype"])
    if s["kind"] == "serve":
        return lib.quantized_linear(s["x"], s["weight_codes"], s["weight_scales"], s["bias"], s["relu"])
    if s["kind"] == "ortho":
        return lib.orthogonalize(s["update"], _STEPS, _COEFFICIENTS)
    lib.muon_step(s["weights"], s["grads"], s["momenta"], _STEP_SIZE, _DECAY, _MOMENTUM, s["nesterov"], _STEPS, _COEFFICIENTS)
    return {"weights": s["weights"], "momenta": s["momenta"]}


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    rows, cols = case["rows"], case["cols"]
    if case["kind"] in ("linear8", "serve"):
        outs = case["outs"]
        token = rows * cols + 4 * rows if case["kind"] == "linear8" else size * rows * cols
        return {"bytes": token + outs * cols + 4 * outs * (2 if case["bias"] else 1) + size * rows * outs,
                "flops": 2 * rows * cols * outs}
    # a step: half of a symmetric product with itself, half of that one's square, one whole product
    short, long = min(rows, cols), max(rows, cols)
    flops = case["count"] * _STEPS * (3 * short * short * long + short ** 3)
    values = case["count"] * rows * cols
    # the update in and out; or weights in and out, momenta (float32) in and out, gradients in
    return {"bytes": values * (2 * size if case["kind"] == "ortho" else 3 * size + 8), "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("linear8", "serve"):
        if case["kind"] == "serve":
            # codes are whole numbers that the definition makes from single-precision values: made here in numpy's
            x = s["x"].float().cpu().numpy()
            scales = np.maximum(np.abs(x).max(axis=1), np.float32(1e-30)) * np.float32(1 / 127)
            codes = np.clip(np.rint(x * (np.float32(1) / scales)[:, None]), -127, 127)
            codes, scales = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
        else:
            codes, scales = s["codes"], s["scales"]
        weight = (s["weight_codes"].double() * s["weight_scales"].double()[:, None]).t().contiguous()
        out = torch.empty((case["rows"], case["outs"]), dtype=torch.float64, device="cuda")
        for r in range(0, case["rows"], 8192):
            part = (codes[r:r + 8192].double() * scales[r:r + 8192].double()[:, None]) @ weight
            if s["bias"] is not None:
                part += s["bias"].double()
            out[r:r + 8192] = torch.relu(part) if s["relu"] else part
        return out

    a, b, c = _COEFFICIENTS

    def orthogonal(u):
        x = u.double()
        x = x / (torch.linalg.matrix_norm(x) + 1e-7)
        for _ in range(_STEPS):
            if x.shape[0] <= x.shape[1]:
                gram = torch.matmul(x, x.t())
                x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
            else:
                gram = torch.matmul(x.t(), x)
                x = a * x + torch.matmul(x, b * gram + c * torch.matmul(gram, gram))
        return x

    if case["kind"] == "ortho":
        u = s["update"]
        return orthogonal(u) if u.dim() == 2 else torch.stack([orthogonal(v) for v in u])
    weights, momenta = [], []
    for w, g, v in zip(s["weights"], s["grads"], s["momenta"]):
        held = _MOMENTUM * v.double() + (1 - _MOMENTUM) * g.double()
        update = _MOMENTUM * held + (1 - _MOMENTUM) * g.double() if case["nesterov"] else held
        weights.append((1 - _DECAY) * w.double() - _STEP_SIZE * orthogonal(update))
        momenta.append(held)
    return {"weights": weights, "momenta": momenta}
