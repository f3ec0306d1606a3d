"""Performance cases of what a training step keeps and learns beside its products: layer norms, activations kept in 8 bits for
the backward pass, and learnt rows.

  * `norm`: layer norm of rows, for serving (`layer_norm`) or with the statistics that training keeps (`layer_norm_train`);
  * `norm_grad`: its gradients, from the rows themselves (`layer_norm_grad`) or from their 8-bit checkpoint
    (`layer_norm_packed_grad`);
  * `store`: activations into a checkpoint and back, `pack_activations` and `unpack_activations`;
  * `linear_grad`: the gradients of a linear layer's weight and bias from the checkpoint of its input, `packed_linear_grad`;
  * `embed`: scaled rows of a table by id, `embedding`;
  * `embed_grad`: the gradient of the table, `embedding_grad`.

A checkpoint has, for each 32 columns of a row, a step that is a power of two, and a code of 8 bits for each value.

`listed()` names twelve cases, `draw()` gives others of the same ranges.  With `own` false `run` computes them from
elementary torch operations in float32, with `own` true it calls the library.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-5
_GROUP = 32


# ---- the cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decoding step: a call whose launch and latency count
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "bfloat16", "train": False},
        # the outputs of a layer for all destination rows of a large block of a graph
        {"name": "norm_block", "kind": "norm", "rows": 250000, "cols": 128, "dtype": "float32", "train": True},
        # a minibatch of 1024 seeds
        {"name": "norm_grad_minibatch", "kind": "norm_grad", "rows": 1024, "cols": 256, "dtype": "float32", "packed": False},
        # a long batch of wide rows
        {"name": "norm_grad_large", "kind": "norm_grad", "rows": 16384, "cols": 8192, "dtype": "bfloat16", "packed": False},
        # a block of a graph with an odd width, from checkpoints
        {"name": "norm_grad_packed_602", "kind": "norm_grad", "rows": 60001, "cols": 602, "dtype": "float32", "packed": True},
        # aggregated features of a large block into a checkpoint and back
        {"name": "store_block", "kind": "store", "rows": 250000, "cols": 100, "dtype": "float32"},
        # the weight of a layer on a minibatch of 1024 seeds
        {"name": "linear_grad_minibatch", "kind": "linear_grad", "rows": 1024, "cols": 128, "outs": 256, "dtype": "float32",
         "bias": True},
        # a first layer over features of an odd width: a long sum for few outputs
        {"name": "linear_grad_602", "kind": "linear_grad", "rows": 60001, "cols": 602, "outs": 128, "dtype": "float32",
         "bias": True},
        # the largest: a long batch through a wide square layer
        {"name": "linear_grad_large", "kind": "linear_grad", "rows": 16384, "cols": 4096, "outs": 4096, "dtype": "bfloat16",
         "bias": False},
        # the learnt rows of the distinct nodes of a block
        {"name": "embed_block", "kind": "embed", "rows": 109074, "table": 2400000, "cols": 100, "dtype": "float32", "hot": False},
        # a minibatch of seeds with ten neighbours each, hot ones among them
        {"name": "embed_grad_minibatch", "kind": "embed_grad", "rows": 11264, "table": 100000, "cols": 128, "dtype": "float32",
         "hot": True},
        # a million ids, of which the hottest is one in ten
        {"name": "embed_grad_large", "kind": "embed_grad", "rows": 1000000, "table": 250000, "cols": 256, "dtype": "bfloat16",
         "hot": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over its logarithm, every other one a whole number of tiles."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 else max(lo, min(hi, (v + 63) // 64 * 64))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "norm_grad", "store", "linear_grad", "linear_grad", "embed", "embed_grad", "embed_grad"])
    case = {"kind": kind, "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"])}
    if kind in ("norm", "norm_grad", "store"):
        cols = _size(rng, 32, 16384)
        # from single rows to long batches, held to 2^27 values
        case.update(rows=_log(rng, 1, min(400000, (1 << 27) // cols)), cols=cols)
        if kind == "norm":
            case.update(train=rng.random() < 0.6)
        elif kind == "norm_grad":
            case.update(packed=rng.random() < 0.5)
    elif kind == "linear_grad":
        cols, outs = _size(rng, 32, 4096), _size(rng, 32, 4096)
        # held to 2^26 values of either operand and a fourth of the largest case's products
        most = min(300000, (1 << 26) // max(cols, outs), (1 << 36) // (cols * outs))
        case.update(rows=_log(rng, 1, most), cols=cols, outs=outs, bias=rng.random() < 0.6)
    else:
        cols = _size(rng, 16, 2048)
        case.update(rows=_log(rng, 1, min(1000000, (1 << 27) // cols)), table=_log(rng, 1000, min(2000000, (1 << 28) // cols)),
                    cols=cols, hot=rng.random() < 0.6)
    return case


# ---- what a caller has in hand ----------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(case, g):
    """Columns of different sizes and offsets, a few of them far larger than the others, rows of different lengths."""
    cols = case["cols"]
    column = torch.exp(0.5 * torch.randn((cols,), generator=g, device="cuda"))
    column[torch.randint(0, cols, (max(1, cols // 200),), generator=g, device="cuda")] *= 8
    offset = 0.3 * torch.randn((cols,), generator=g, device="cuda")
    length = torch.exp(0.3 * torch.randn((case["rows"], 1), generator=g, device="cuda"))
    return torch.randn((case["rows"], cols), generator=g, device="cuda").add_(offset).mul_(length).mul_(column)


def _gradients(rows, cols, g):
    """Rows of different sizes, one in fifty of them zero: positions that a loss leaves out."""
    size = torch.exp(torch.randn((rows, 1), generator=g, device="cuda")) * 1e-3
    size[torch.rand((rows, 1), generator=g, device="cuda") < 0.02] = 0
    return torch.randn((rows, cols), generator=g, device="cuda").mul_(size)


def _codes(x):
    """float32 x [rows, cols] -> (codes int8 in rows of whole 16 bytes, exponents uint8): code * 2^(exponent - 127)."""
    rows, cols = x.shape
    groups = (cols + _GROUP - 1) // _GROUP
    whole = torch.nn.functional.pad(x, (0, groups * _GROUP - cols)).view(rows, groups, _GROUP)
    # the least power of two of which 127 reach the largest value: 127 = 1.984375 * 2^6
    most = whole.abs().amax(dim=2).view(torch.int32)
    exponents = torch.clamp(((most + 0x1FFFF) >> 23) - 6, min=1)
    least = ((254 - exponents) << 23).view(torch.float32)
    codes = torch.round(whole * least[..., None]).view(rows, groups * _GROUP)
    room = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    room[:, :cols] = codes[:, :cols]
    return room[:, :cols], exponents.to(torch.uint8)


def _ids(case, g):
    n, table = case["rows"], case["table"]
    if not case["hot"]:
        ids = torch.randint(0, table, (n,), generator=g, device="cuda")
        return ids if n > table else torch.sort(ids).values           # (a block's nodes, as a relabelling leaves them)
    # density x^-1.1 over the table, the hot ones spread over it, and places of a padded batch
    u = torch.rand((n,), generator=g, device="cuda", dtype=torch.float64)
    rank = ((1 + u * (float(table + 1) ** -0.1 - 1)) ** -10.0).long().clamp_(1, table) - 1
    ids = (rank * 7919 + 13) % table
    return torch.where(torch.rand((n,), generator=g, device="cuda") < 0.02, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    dtype = state["type"] = _DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        x = _activations(case, g).to(dtype)
        state["weight"] = (1 + 0.2 * torch.randn((case["cols"],), generator=g, device="cuda")).to(dtype)
        state["bias"] = (0.2 * torch.randn((case["cols"],), generator=g, device="cuda")).to(dtype)
        if kind == "norm":
            state["x"] = x
            return state
        state["grad"] = _gradients(case["rows"], case["cols"], g).to(dtype)
        wide = x.float()
        state["mean"] = wide.mean(dim=1)
        state["rstd"] = torch.rsqrt((wide - state["mean"][:, None]).square().mean(dim=1) + _EPS)
        if case["packed"]:
            state["codes"], state["exponents"] = _codes(wide)
        else:
            state["x"] = x
    elif kind == "store":
        state["x"] = _activations(case, g).to(dtype)
    elif kind == "linear_grad":
        state["codes"], state["exponents"] = _codes(torch.relu(_activations(case, g)))
        state["grad"] = _gradients(case["rows"], case["outs"], g).to(dtype)
    else:
        state["ids"] = _ids(case, g)
        if kind == "embed":
            state["rows_of"] = torch.randn((case["table"], case["cols"]), generator=g, device="cuda").to(dtype)
        else:
            state["grad"] = _gradients(case["rows"], case["cols"], g).to(dtype)
        state["scale"] = math.sqrt(case["cols"])
    return state


# ---- one pass ---------------------------------------------------------------------------------------
def _decoded(codes, exponents):
    cols = codes.shape[1]
    step = (exponents.to(torch.int32) << 23).view(torch.float32).repeat_interleave(_GROUP, dim=1)[:, :cols]
    return codes.float() * step


def _plain(s):
    kind, dtype = s["kind"], s["type"]
    if kind == "norm":
        x = s["x"].float()
        mean = x.mean(dim=1)
        apart = x - mean[:, None]
        rstd = torch.rsqrt(apart.square().mean(dim=1) + _EPS)
        out = (apart * rstd[:, None] * s["weight"].float() + s["bias"].float()).to(dtype)
        return (out, mean, rstd) if s["train"] else out
    if kind == "norm_grad":
        x = _decoded(s["codes"], s["exponents"]) if s["packed"] else s["x"].float()
        grad, rstd = s["grad"].float(), s["rstd"][:, None]
        unit = (x - s["mean"][:, None]) * rstd
        part = grad * s["weight"].float()
        dx = rstd * (part - part.mean(dim=1, keepdim=True) - unit * (part * unit).mean(dim=1, keepdim=True))
        return dx.to(dtype), (grad * unit).sum(dim=0).to(dtype), grad.sum(dim=0).to(dtype)
    if kind == "store":
        return _decoded(*_codes(s["x"].float())).to(dtype)
    if kind == "linear_grad":
        grad = s["grad"].float()
        weight = (grad.t() @ _decoded(s["codes"], s["exponents"])).to(dtype)
        return (weight, grad.sum(dim=0).to(dtype)) if s["bias"] else weight
    ids = s["ids"]
    inside = (ids >= 0) & (ids < s["table"])
    held = torch.where(inside, ids, torch.zeros_like(ids))
    if kind == "embed":
        return (s["rows_of"][held].float() * s["scale"] * inside[:, None]).to(dtype)
    table = torch.zeros((s["table"], s["cols"]), device=ids.device)
    table.index_add_(0, held, s["grad"].float() * inside[:, None])
    return (table * s["scale"]).to(dtype)


def run(state):
    s = state
    if not own:
        return _plain(s)
    import f2cgt_amd
    lib = f2cgt_amd.load()
    kind = s["kind"]
    if kind == "norm":
        if s["train"]:
            return lib.layer_norm_train(s["x"], s["weight"], s["bias"], _EPS)
        return lib.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    if kind == "norm_grad":
        if s["packed"]:
            return lib.layer_norm_packed_grad(s["grad"], s["codes"], s["exponents"], s["mean"], s["rstd"], s["weight"])
        return lib.layer_norm_grad(s["grad"], s["x"], s["mean"], s["rstd"], s["weight"])
    if kind == "store":
        codes, exponents = lib.pack_activations(s["x"])
        return lib.unpack_activations(codes, exponents, s["type"])
    if kind == "linear_grad":
        weight, bias = lib.packed_linear_grad(s["grad"], s["codes"], s["exponents"], s["bias"], s["type"])
        return (weight, bias) if s["bias"] else weight
    if kind == "embed":
        return lib.embedding(s["rows_of"], s["ids"], s["scale"])
    return lib.embedding_grad(s["grad"], s["ids"], s["table"], s["scale"])


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    values = rows * cols
    kept = values + rows * ((cols + _GROUP - 1) // _GROUP)            # bytes of a checkpoint
    if kind == "norm":
        return {"bytes": 2 * size * values + 2 * size * cols + (8 * rows if case["train"] else 0), "flops": 8 * values}
    if kind == "norm_grad":
        return {"bytes": 2 * size * values + (kept if case["packed"] else size * values) + 8 * rows + 3 * size * cols,
                "flops": 14 * values}
    if kind == "store":
        return {"bytes": 2 * size * values + 2 * kept, "flops": 4 * values}
    if kind == "linear_grad":
        outs = case["outs"]
        return {"bytes": size * rows * outs + kept + size * outs * (cols + (1 if case["bias"] else 0)),
                "flops": 2 * rows * cols * outs}
    if kind == "embed":
        return {"bytes": 2 * size * values + 8 * rows, "flops": values}
    return {"bytes": size * (values + case["table"] * cols) + 8 * rows, "flops": values}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def _two_to(e):
    """2^e in float64 of whole numbers e, from its bits (a power by way of a logarithm is not exact)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_step(most):
    """The step of a group whose largest size is `most` (float64): the least 2^e, e >= -126, with most <= 127 * 2^e."""
    fraction, power = torch.frexp(most)
    e = torch.where(fraction > 127 / 128, power - 6, power - 7)
    return _two_to(torch.clamp(e, min=-126))


def _exact_values(codes, exponents):
    out = codes.double()
    for j in range(exponents.shape[1]):
        part = out[:, j * _GROUP:(j + 1) * _GROUP]
        part *= _two_to(exponents[:, j:j + 1].long() - 127)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + _EPS)
        out = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], s["weight"].double())
        return (out, mean, rstd) if case["train"] else out
    if kind == "norm_grad":
        x = _exact_values(s["codes"], s["exponents"]) if case["packed"] else s["x"].double()
        grad = s["grad"].double()
        mean, rstd, weight = s["mean"].double(), s["rstd"].double(), s["weight"].double()
        # n = r (x - mean); dx = r (g w - n (n . g w) / d - sum(g w) / d)
        x -= mean[:, None]
        x *= rstd[:, None]
        along = (grad * x)
        dw, db = along.sum(dim=0), grad.sum(dim=0)
        second = torch.mv(along, weight) / case["cols"]
        first = torch.mv(grad, weight) / case["cols"]
        del along
        grad *= weight
        grad -= first[:, None]
        grad -= x * second[:, None]
        return grad * rstd[:, None], dw, db
    if kind == "store":
        x = s["x"].double()
        for c in range(0, case["cols"], _GROUP):
            part = x[:, c:c + _GROUP]
            step = _exact_step(part.abs().amax(dim=1, keepdim=True))
            part.copy_(torch.round(part / step) * step)
        return x
    if kind == "linear_grad":
        values, grad = _exact_values(s["codes"], s["exponents"]), s["grad"].double()
        weight = torch.mm(grad.t(), values)
        return (weight, grad.sum(dim=0)) if case["bias"] else weight
    ids = s["ids"]
    keep = torch.nonzero((ids >= 0) & (ids < case["table"])).flatten()
    if kind == "embed":
        out = torch.zeros((case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
        out[keep] = s["rows_of"].index_select(0, ids[keep]).double() * s["scale"]
        return out
    table = torch.zeros((case["table"], case["cols"]), dtype=torch.float64, device="cuda")
    for r in range(0, keep.numel(), 1 << 18):
        at = keep[r:r + (1 << 18)]
        table.index_add_(0, ids[at], s["grad"][at].double() * s["scale"])
    return table
