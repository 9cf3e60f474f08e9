"""The operators of the training head over an embedding table, as a user's program calls them, with their plain forms.

A ranking or retrieval model takes the looked-up rows of a batch, drops out and normalises them, and scores the result
against every row of an item table; the loss is the softmax cross entropy over that table and its gradient goes back
into the rows.  Three operators, each with its backward pass:

  layer_norm    y = (x - mean) * rstd * weight + bias over the last dimension
  dropout       y = x * keep / P(keep), keep from a counter-based generator, the mask stored nowhere
  softmax_loss  loss_n = log sum_v exp(z_nv) - z_n,target(n),  z_nv = scale * x_n . table_v + item_bias_v

`run` makes the framework's calls where `own` is true and computes the same from elementary torch operations elsewhere.
"""
import math

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_MASKED_BELOW = -1e30   # an item_bias at or below this takes the item out of the softmax


def listed():
    return [
        # normalising the concatenated lookup of a pooled-embedding batch: 16384 samples, 26 features of 64 columns
        {"name": "norm_train_bf16_1664", "op": "norm", "train": True, "rows": 16384, "dim": 1664, "type": "bf16", "wtype": "f32"},
        # one small table's rows, 4096 keys a step: latency counts
        {"name": "norm_train_f32_small", "op": "norm", "train": True, "rows": 4096, "dim": 16, "type": "f32", "wtype": "f32"},
        # the 128-column rows of a ranking batch of 65536, all 26 features
        {"name": "norm_train_f32_128", "op": "norm", "train": True, "rows": 1703936, "dim": 128, "type": "f32", "wtype": "f32"},
        # evaluation with an odd width, half precision
        {"name": "norm_eval_f16_odd", "op": "norm", "train": False, "rows": 30011, "dim": 1001, "type": "f16", "wtype": "f16"},
        # dropout on the float32 lookup of a ranking batch (65536 samples, 26 features of 128), forward and backward
        {"name": "drop_train_f32_large", "op": "drop", "train": True, "rows": 65536, "dim": 3328, "type": "f32", "p": 0.1},
        # the same between bfloat16 layers of a pooled batch
        {"name": "drop_train_bf16", "op": "drop", "train": True, "rows": 16384, "dim": 1664, "type": "bf16", "p": 0.25},
        # evaluation: the scores' normaliser of a few queries against a whole item table: bound by reading the table
        {"name": "loss_eval_bf16_one", "op": "loss", "train": False, "rows": 1, "items": 1000000, "dim": 64, "type": "bf16", "biased": False},
        # in-batch softmax: the distinct items of a batch are the vocabulary, float32 rows as the lookup returns them
        {"name": "loss_train_f32_batch", "op": "loss", "train": True, "rows": 4096, "items": 3911, "dim": 64, "type": "f32", "biased": True},
        # training against a table of 1 M items
        {"name": "loss_train_bf16_1m", "op": "loss", "train": True, "rows": 2048, "items": 1000000, "dim": 128, "type": "bf16", "biased": False},
        # training with popularity corrections and free slots, many rows, 64 columns
        {"name": "loss_train_bf16_64", "op": "loss", "train": True, "rows": 8192, "items": 200003, "dim": 64, "type": "bf16", "biased": True},
        # float32 table
        {"name": "loss_train_f32_128", "op": "loss", "train": True, "rows": 1024, "items": 100000, "dim": 128, "type": "f32", "biased": False},
        # odd sizes: columns that are no multiple of anything, a ragged item count
        {"name": "loss_train_bf16_odd", "op": "loss", "train": True, "rows": 301, "items": 30011, "dim": 201, "type": "bf16", "biased": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "drop", "loss", "loss"])
    train = rng.random() < 0.7
    if op == "loss":
        dim = _log_int(rng, 1, 256)
        items = _log_int(rng, 64, 1000000)
        most = min(16384, 2.6e11 / (dim * items), 2.0e9 / items)   # no more than the largest listed case
        rows = _log_int(rng, 1, max(1, most))
        return {"op": op, "train": train, "rows": rows, "items": items, "dim": dim, "type": rng.choice(["f32", "bf16", "bf16"]),
                "biased": rng.random() < 0.5}
    dim = _log_int(rng, 12, 8192)   # the repository's narrowest rows have 16 columns
    rows = _log_int(rng, 1, min(1703936, 2.0e8 / dim))
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        return {"op": op, "train": train, "rows": rows, "dim": dim, "type": kind, "wtype": rng.choice([kind, "f32"])}
    return {"op": op, "train": train, "rows": rows, "dim": dim, "type": kind, "p": round(rng.uniform(0.02, 0.6), 3)}


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    kind = _TYPES[case["type"]]
    rows, dim = case["rows"], case["dim"]

    def normal(*shape, std=1.0, to=kind):
        return (torch.randn(*shape, generator=g, device=_DEV) * std).to(to)

    state = {"case": case}
    if case["op"] == "norm":
        weight = _TYPES[case["wtype"]]
        # columns with offsets of their own, as rows of different features have
        state["x"] = (torch.randn(rows, dim, generator=g, device=_DEV) * 0.5 + torch.randn(1, dim, generator=g, device=_DEV)).to(kind)
        state["weight"] = (1 + 0.1 * torch.randn(dim, generator=g, device=_DEV)).to(weight)
        state["bias"] = normal(dim, std=0.1, to=weight)
        state["eps"] = 1e-5
        if case["train"]:
            state["grad"] = normal(rows, dim, std=1e-2)
    elif case["op"] == "drop":
        state["x"] = normal(rows, dim)
        state["seed"], state["offset"] = 1234567 + 7919 * seed, seed * (1 << 33) + 5
        if case["train"]:
            state["grad"] = normal(rows, dim, std=1e-2)
    else:
        items = case["items"]
        state["x"] = normal(rows, dim)
        state["table"] = normal(items, dim, std=0.5)
        state["scale"] = 4.0 / math.sqrt(dim)
        state["bias"] = None
        target = torch.randint(0, items, (rows,), generator=g, device=_DEV)
        if case["biased"]:
            # minus the log of each item's frequency; about 1 slot in 20 of the table is free
            bias = 0.5 * torch.randn(items, generator=g, device=_DEV) + 1
            free = torch.rand(items, generator=g, device=_DEV) < 0.05
            free[0] = False
            state["bias"] = torch.where(free, torch.full_like(bias, -math.inf), bias)
            target = torch.where(free[target], torch.zeros_like(target), target)
        # about 1 position in 16 is padding: no target
        pad = torch.rand(rows, generator=g, device=_DEV) < 1 / 16
        pad[0] = False
        state["target"] = torch.where(pad, torch.full_like(target, -1), target)
        if case["train"]:
            # the mean over the positions, weighted
            state["grad"] = (0.5 + torch.rand(rows, generator=g, device=_DEV)) / rows
    return state


def _ops():
    from recsdk_amd import torch_ops

    torch_ops.load()
    return torch.ops.recsdk


def run(state):
    op, train = state["case"]["op"], state["case"]["train"]
    if own:
        ops = _ops()
        x = state["x"].detach().requires_grad_(train)
        if op == "norm":
            weight, bias = (state[k].detach().requires_grad_(train) for k in ("weight", "bias"))
            y = ops.layer_norm(x, weight, bias, state["eps"])
            return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), state["grad"])) if train else y
        if op == "drop":
            y = ops.dropout(x, state["case"]["p"], state["seed"], state["offset"])
            return (y.detach(), *torch.autograd.grad(y, (x,), state["grad"])) if train else y
        table = state["table"].detach().requires_grad_(train)
        loss = ops.softmax_loss(x, table, state["target"], state["bias"], state["scale"])
        return (loss.detach(), *torch.autograd.grad(loss, (x, table), state["grad"])) if train else loss
    with torch.no_grad():
        return {"norm": _norm, "drop": _drop, "loss": _loss}[op](state, train)


# ---- plain forms --------------------------------------------------------------------------------------------------


def _norm(state, train):
    x, weight = state["x"].float(), state["weight"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + state["eps"])
    hat = centred * rstd
    y = (hat * weight + state["bias"].float()).to(state["x"].dtype)
    if not train:
        return y
    grad = state["grad"].float()
    dhat = grad * weight
    dx = rstd * (dhat - dhat.mean(1, keepdim=True) - hat * (dhat * hat).mean(1, keepdim=True))
    return y, dx.to(state["x"].dtype), (grad * hat).sum(0).to(state["weight"].dtype), grad.sum(0).to(state["bias"].dtype)


def _round(c, key):
    """One round of Philox-4x32 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011)."""
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # 64-bit products; int64 wraps to the same bits
    m = 0xFFFFFFFF
    return ((b >> 32) & m) ^ c[1] ^ key[0], b & m, ((a >> 32) & m) ^ c[3] ^ key[1], a & m


def _kept(count, p, seed, offset):
    """Truth value per element: element e takes 16 bits, number e % 8 of the block with counter (e // 8, offset) under
    the key `seed`, and is kept where they are below round(65536 (1 - p))."""
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=_DEV)
    m = 0xFFFFFFFF
    c = (block & m, block >> 32, torch.full_like(block, offset & m), torch.full_like(block, (offset >> 32) & m))
    k0, k1 = seed & m, (seed >> 32) & m
    for r in range(10):
        c = _round(c, ((k0 + r * 0x9E3779B9) & m, (k1 + r * 0xBB67AE85) & m))
    words = torch.stack(c, 1)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:count]
    below = round(65536 * (1 - p))
    return halves < below, 65536 / below


def _drop(state, train):
    x = state["x"]
    keep, factor = _kept(x.numel(), state["case"]["p"], state["seed"], state["offset"])
    keep = keep.reshape(x.shape)
    zero = torch.zeros((), device=_DEV)
    y = torch.where(keep, x.float() * factor, zero).to(x.dtype)
    return (y, torch.where(keep, state["grad"].float() * factor, zero).to(x.dtype)) if train else y


def _loss(state, train):
    x, table, target, scale = state["x"].float(), state["table"].float(), state["target"], state["scale"]
    items = table.shape[0]
    live = (target >= 0) & (target < items)
    at = torch.where(live, target, torch.zeros_like(target))
    logits = x @ table.t()
    logits *= scale
    if state["bias"] is not None:
        logits += torch.where(state["bias"] <= _MASKED_BELOW, torch.full_like(state["bias"], -math.inf), state["bias"])
    top = logits.amax(1, keepdim=True)
    mine = logits.gather(1, at[:, None])
    logits -= top
    logits.exp_()
    total = logits.sum(1, keepdim=True)
    loss = (total.log() + top - mine)[:, 0]
    loss = torch.where(live, loss, torch.zeros_like(loss))
    if not train:
        return loss
    logits /= total
    logits.scatter_add_(1, at[:, None], torch.full_like(mine, -1))
    logits *= torch.where(live, state["grad"] * scale, torch.zeros_like(loss))[:, None]
    return loss, (logits @ table).to(state["x"].dtype), (logits.t() @ x).to(state["table"].dtype)


# ---- the operators' definitions in 64 bits ------------------------------------------------------------------------


def _exact_norm(state, train):
    x, w, b = state["x"].double(), state["weight"].double(), state["bias"].double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    hat = (x - mean) / (var + state["eps"]).sqrt()
    if not train:
        return hat * w + b
    g = state["grad"].double()
    gw = g * w
    # (I - 11'/D - hat hat'/D) gw / sigma
    dx = (gw - gw.sum(1, keepdim=True) / x.shape[1] - hat * (gw * hat).sum(1, keepdim=True) / x.shape[1]) / (var + state["eps"]).sqrt()
    return hat * w + b, dx, torch.einsum("nd,nd->d", g, hat), g.sum(0)


def _exact_drop(state, train):
    import numpy as np

    # numpy's unsigned integers: the generator written apart from the plain form's
    n, p = state["x"].numel(), state["case"]["p"]
    if n > 40000000:
        return None
    c = np.zeros((4, (n + 7) // 8), dtype=np.uint64)
    m = np.uint64(0xFFFFFFFF)
    c[0] = np.arange(c.shape[1], dtype=np.uint64)
    c[2], c[3] = state["offset"] % (1 << 32), (state["offset"] >> 32) % (1 << 32)
    key = [state["seed"] % (1 << 32), (state["seed"] >> 32) % (1 << 32)]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), p0 & m])
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    bits = np.ascontiguousarray(c.T.astype("<u4")).view("<u2").reshape(-1)[:n].astype(np.int64)
    below = round(65536 * (1 - p))
    factor = torch.from_numpy(np.where(bits < below, 65536.0 / below, 0.0)).to(_DEV).reshape(state["x"].shape)
    y = state["x"].double() * factor
    return (y, state["grad"].double() * factor) if train else y


def _exact_loss(state, train):
    x, table = state["x"].double(), state["table"].double()
    rows, items = x.shape[0], table.shape[0]
    bias = torch.zeros(items, device=_DEV, dtype=torch.float64) if state["bias"] is None else state["bias"].double()
    loss = torch.zeros(rows, device=_DEV, dtype=torch.float64)
    dx, dtable = torch.zeros_like(x), torch.zeros_like(table)
    step = max(1, 400000000 // items)   # rows at a time
    for lo in range(0, rows, step):
        part, t = x[lo:lo + step], state["target"][lo:lo + step]
        z = state["scale"] * torch.mm(part, table.T) + bias
        z.masked_fill_((bias <= _MASKED_BELOW)[None], -math.inf)
        norm = torch.logsumexp(z, 1)
        row = torch.arange(part.shape[0], device=_DEV)
        on = (t >= 0).double()
        loss[lo:lo + step] = on * (norm - z[row, t.clamp(min=0)])
        if train:
            z.sub_(norm[:, None]).exp_()
            z[row, t.clamp(min=0)] -= 1
            z *= (on * state["grad"][lo:lo + step].double() * state["scale"])[:, None]
            dx[lo:lo + step] = torch.mm(z, table)
            dtable += torch.mm(z.T, part)
    return (loss, dx, dtable) if train else loss


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "drop": _exact_drop, "loss": _exact_loss}[case["op"]](state, case["train"])


def work(case):
    rows, dim, train = case["rows"], case["dim"], case["train"]
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    n = rows * dim
    if case["op"] == "norm":
        wsize = {"f32": 4, "bf16": 2, "f16": 2}[case["wtype"]]
        # forward: x, y; backward: the gradient and dx (x once over both)
        return {"bytes": n * size * (4 if train else 2) + dim * wsize * (4 if train else 2), "flops": n * (16 if train else 8)}
    if case["op"] == "drop":
        return {"bytes": n * size * (4 if train else 2), "flops": n * (2 if train else 1)}
    items = case["items"]
    fixed = rows * 12 + (4 * items if case["biased"] else 0)
    if not train:
        return {"bytes": (n + items * dim) * size + fixed, "flops": 2 * rows * items * dim}
    return {"bytes": 2 * (n + items * dim) * size + fixed + 4 * rows, "flops": 6 * rows * items * dim}
