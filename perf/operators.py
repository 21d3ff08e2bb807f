"""The residual-path operators of the pair stack, as cases to be timed and checked.

Between two pair layers a training step computes

    dropout_add             z' = z + m * y / (1 - p)          m: keep mask from a counter-based generator
    layer_norm              h  = (z' - mean) * rstd * w + b   over the channels of each pair
    dropout_add_layer_norm  both in one pass

and their gradients.  `run` computes one of them: with `own` false from elementary torch operations in 32 bits,
with `own` true through the framework.  `exact` gives the same values from the definitions in 64 bits.

The keep mask is a function of (seed, offset, position) alone: position m of the mask tensor takes word m mod 4 of
Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011) with the key = seed and
the counter = (m div 4, offset), and is dropped if that word is below p * 2^32.  `share` names the axes along which
one draw is shared (the mask has size 1 there).  The factor 1 / (1 - p) is a number of 32 bits, z' is rounded to 32 bits
and from there to the stream's type, and the norm that follows is taken of z' as it is held.
"""

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
# Axes of [B, I, J, C] that share one draw: "row" is one draw for each row i of the pair tensor, "column" one for each
# column j, "row_channel" one for each column and channel (shared by the rows), "element" one for each value.
SHARE = {"row": (2, 3), "column": (1, 3), "row_channel": (1,), "element": ()}
EPS = 1e-5
LOW = 0xFFFFFFFF


def listed():
    def c(name, op, train, b, i, j, dim, z, y, out, share="", p=0.0, swap=False):
        return {"name": name, "op": op, "train": train, "b": b, "i": i, "j": j, "dim": dim, "z": z, "y": y,
                "out": out, "share": share, "p": p, "swap": swap}

    return [
        # the 16-bit LayerNorm input of an attention layer over a very small complex: a call's latency
        c("ln_n9", "layer_norm", False, 1, 9, 9, 128, "float32", "", "bfloat16"),
        # the same at the benchmark's size for an ending node: read with the pair's axes swapped
        c("ln_swapped_n1024", "layer_norm", False, 1, 1024, 1024, 128, "float32", "", "bfloat16", swap=True),
        # training in fp32 at the smaller benchmark size
        c("ln_train_n384", "layer_norm", True, 1, 384, 384, 128, "float32", "", "float32"),
        # training with wide rows, all in 16 bits
        c("ln_train_wide", "layer_norm", True, 1, 1, 8192, 4096, "bfloat16", "", "bfloat16"),
        # ragged: an odd number of channels, so that no row but every eighth starts on a 16-byte boundary
        c("ln_train_odd", "layer_norm", True, 2, 33, 129, 333, "float16", "", "float16"),
        # the recycling passes of a training step: dropout on, no gradient, the benchmark's size
        c("drop_row_n1024", "dropout_add", False, 1, 1024, 1024, 128, "float32", "float32", "", "row", 0.25),
        # ordinary dropout on a token stream, with the update's gradient
        c("drop_element_train", "dropout_add", True, 1, 1, 16384, 1024, "bfloat16", "bfloat16", "", "element", 0.1),
        # the ending node's shared mask, a 16-bit update onto an fp32 stream
        c("drop_column_train_n200", "dropout_add", True, 1, 200, 200, 128, "float32", "bfloat16", "", "column", 0.25),
        # smallest training step of the fused operator: latency
        c("fused_train_n9", "dropout_add_layer_norm", True, 1, 9, 9, 128, "float32", "float32", "float32", "row", 0.25),
        # the pair block's hand-over between two layers at the benchmark's size
        c("fused_row_n1024", "dropout_add_layer_norm", False, 1, 1024, 1024, 128, "float32", "float32", "bfloat16", "row",
          0.25),
        # the same in training at the deep stack's size, after an ending node
        c("fused_column_train_n768", "dropout_add_layer_norm", True, 1, 768, 768, 128, "float32", "float32", "bfloat16",
          "column", 0.25),
        # a 16-bit residual stream of tokens
        c("fused_element_train", "dropout_add_layer_norm", True, 1, 2, 4099, 1024, "float16", "float16", "float16",
          "element", 0.1),
    ]


def draw(rng):
    op = rng.choice(["layer_norm", "dropout_add", "dropout_add_layer_norm"])
    dim = rng.choice([128, 128, int(round(2 ** rng.uniform(3, 13))), int(round(2 ** rng.uniform(0, 10))) * 8])
    dim = min(dim, 8192)
    most = 2 ** 26 // dim
    rows = max(1, int(2 ** rng.uniform(0, 20)))
    rows = min(rows, most)
    b = rng.choice([1, 1, 2, 3]) if rows >= 16 else 1
    i = max(1, int(round((rows / b) ** rng.uniform(0.0, 0.6))))
    j = max(1, rows // (b * i))
    z, out = rng.choice([("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"),
                         ("bfloat16", "bfloat16"), ("float16", "float16")])
    y = z if z != "float32" else rng.choice(["float32", out])
    drops = op != "layer_norm"
    return {"op": op, "train": rng.random() < 0.6, "b": b, "i": i, "j": j, "dim": dim, "z": z,
            "y": y if drops else "", "out": out if op != "dropout_add" else "",
            "share": rng.choice(["row", "column", "row_channel", "element"]) if drops else "",
            "p": round(rng.uniform(0.02, 0.6), 3) if drops else 0.0,
            "swap": op == "layer_norm" and rng.random() < 0.3}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape, dim, train = (case["b"], case["i"], case["j"], case["dim"]), case["dim"], case["train"]

    def normal(size, kind="float32"):
        return torch.randn(size, generator=g, device="cuda", dtype=torch.float32).to(TYPES[kind])

    state = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15 + 1) & (2 ** 63 - 1), "offset": seed % 1000}
    # a residual stream: channels with means and spreads of their own
    z = torch.randn(shape, generator=g, device="cuda").mul_(0.5 + normal((dim,)).abs()).add_(normal((dim,)))
    z = z.to(TYPES[case["z"]])
    if case["swap"]:
        z = z.transpose(1, 2)
    state["z"] = z.requires_grad_(train)
    if case["op"] != "layer_norm":
        state["y"] = normal(shape, case["y"]).requires_grad_(train)
        if train:
            state["dz"] = normal(shape, case["z"])
    if case["op"] != "dropout_add":
        state["w"] = normal((dim,)).mul_(0.1).add_(1.0).requires_grad_(train)
        state["b"] = normal((dim,)).mul_(0.1).requires_grad_(train)
        if train:
            state["dh"] = normal(z.shape, case["out"])
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from boltz_mlx_b200 import dropout_add, dropout_add_layer_norm, layer_norm

    case, z = state["case"], state["z"]
    if case["op"] == "layer_norm":
        h = layer_norm(z, state["w"], state["b"], EPS, out_dtype=TYPES[case["out"]])
        if not case["train"]:
            return {"h": h}
        dz, dw, db = torch.autograd.grad(h, (z, state["w"], state["b"]), state["dh"])
        return {"h": h, "dz": dz, "dw": dw, "db": db}
    y, share = state["y"], SHARE[case["share"]]
    if case["op"] == "dropout_add":
        s = dropout_add(z, y, case["p"], state["seed"], state["offset"], share=share)
        if not case["train"]:
            return {"s": s}
        dz, dy = torch.autograd.grad(s, (z, y), state["dz"])
        return {"s": s, "dz": dz, "dy": dy}
    s, h = dropout_add_layer_norm(z, y, state["w"], state["b"], case["p"], state["seed"], state["offset"], share=share,
                                  eps=EPS, out_dtype=TYPES[case["out"]])
    if not case["train"]:
        return {"s": s, "h": h}
    dz, dy, dw, db = torch.autograd.grad((s, h), (z, y, state["w"], state["b"]), (state["dz"], state["dh"]))
    return {"s": s, "h": h, "dz": dz, "dy": dy, "dw": dw, "db": db}


# ---- the plain forms ---------------------------------------------------------------------------------
def _words(count, seed, offset, device):
    """The first `count` 32-bit words of the generator, as int64 (a product of two 32-bit numbers wraps there, and
    its upper half is taken with a mask)."""
    block = torch.arange((count + 3) // 4, device=device)
    c0, c1 = block & LOW, block >> 32
    c2, c3 = torch.full_like(block, offset & LOW), torch.full_like(block, offset >> 32)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack((c0, c1, c2, c3), -1).reshape(-1)[:count]


def _keep(state):
    case, shape = state["case"], list(state["z"].shape)
    for axis in SHARE[case["share"]]:
        shape[axis] = 1
    count = shape[0] * shape[1] * shape[2] * shape[3]
    words = _words(count, state["seed"], state["offset"], state["z"].device)
    return (words >= int(case["p"] * 2.0 ** 32 + 0.5)).reshape(shape)


def _norm(x, w, b):
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = ((centred * centred).mean(-1, keepdim=True) + EPS).rsqrt()
    hat = centred * rstd
    return hat * w + b, hat, rstd


def _norm_gradients(dh, hat, rstd, w):
    g = dh * w
    dx = (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True)) * rstd
    return dx, (dh * hat).sum((0, 1, 2)), dh.sum((0, 1, 2))


def _run_plain(state):
    case = state["case"]
    with torch.no_grad():
        z = state["z"].detach()
        if case["op"] == "layer_norm":
            h, hat, rstd = _norm(z.float(), state["w"], state["b"])
            r = {"h": h.to(TYPES[case["out"]])}
            if case["train"]:
                dx, r["dw"], r["db"] = _norm_gradients(state["dh"].float(), hat, rstd, state["w"])
                r["dz"] = dx.to(z.dtype)
            return r
        keep, scale = _keep(state), 1.0 / (1.0 - case["p"])
        y = state["y"].detach()
        # A stream held in 16 bits is summed in 64: a value next to the border between two of its steps would fall to
        # the other side by the rounding of the product, and move the norm of the whole row with it.
        wide = torch.float32 if z.dtype == torch.float32 else torch.float64
        factor = torch.full((), scale, dtype=torch.float32, device=z.device).to(wide)
        s = (z.to(wide) + torch.where(keep, y.to(wide) * factor, 0.0)).float().to(z.dtype)
        r = {"s": s}
        if case["op"] == "dropout_add":
            if case["train"]:
                r["dz"] = state["dz"]
                r["dy"] = torch.where(keep, state["dz"].float() * scale, 0.0).to(y.dtype)
            return r
        h, hat, rstd = _norm(s.float(), state["w"], state["b"])
        r["h"] = h.to(TYPES[case["out"]])
        if case["train"]:
            dx, r["dw"], r["db"] = _norm_gradients(state["dh"].float(), hat, rstd, state["w"])
            ds = dx + state["dz"].float()
            r["dz"] = ds.to(z.dtype)
            r["dy"] = torch.where(keep, ds * scale, 0.0).to(y.dtype)
        return r


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    rows = case["b"] * case["i"] * case["j"]
    n = rows * case["dim"]
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "": 0}
    z, y, out = size[case["z"]], size[case["y"]], size[case["out"]]
    params = 8 * case["dim"]
    if case["op"] == "layer_norm":
        return {"bytes": n * (z + out) * (2 if case["train"] else 1) + params * (2 if case["train"] else 1),
                "flops": n * (25 if case["train"] else 9)}
    if case["op"] == "dropout_add":
        # the stream's gradient is the given one, untouched
        return {"bytes": n * (2 * z + y + (z + y if case["train"] else 0)), "flops": n * (3 if case["train"] else 2)}
    if case["train"]:  # z, y, dz, dh in; s, h, dz, dy out
        return {"bytes": n * (4 * z + 2 * y + 2 * out) + 2 * params, "flops": n * 30}
    return {"bytes": n * (2 * z + y + out) + params, "flops": n * 11}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _exact_keep(case, seed, offset):
    """The keep mask as a boolean array, from unsigned 64-bit products."""
    shape = [1 if axis in SHARE[case["share"]] else case[k] for axis, k in enumerate(("b", "i", "j", "dim"))]
    count = int(np.prod(shape))
    m = np.arange(-(-count // 4), dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    x = [m & low, m >> half, np.full_like(m, offset & LOW), np.full_like(m, offset >> 32)]
    key = [seed & LOW, seed >> 32]
    for n in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        r0, r1 = np.uint64((key[0] + n * 0x9E3779B9) & LOW), np.uint64((key[1] + n * 0xBB67AE85) & LOW)
        x = [(q >> half) ^ x[1] ^ r0, q & low, (p >> half) ^ x[3] ^ r1, p & low]
    words = np.stack(x, 1).ravel()[:count]
    return torch.from_numpy(words >= np.uint64(int(case["p"] * 2.0 ** 32 + 0.5))).reshape(shape).cuda()


def exact(case, seed):
    state = prepare(dict(case), seed)
    train, wide = case["train"], {}
    for k in ("z", "y", "w", "b"):
        if k in state:
            wide[k] = state[k].detach().double().requires_grad_(train)
    s, r, heads, grads = wide["z"], {}, [], []
    with torch.set_grad_enabled(train):
        if case["op"] != "layer_norm":
            factor = float(np.float32(1.0 / (1.0 - case["p"])))
            s = s + wide["y"] * (_exact_keep(case, state["seed"], state["offset"]).double() * factor)
            r["s"] = s.detach()
            heads, grads = [s], [state["dz"].double()] if train else []
        if case["op"] != "dropout_add":
            if case["op"] != "layer_norm":  # the norm is taken of the stream as it is held
                s = s + (s.detach().float().to(TYPES[case["z"]]).double() - s.detach())
            n = case["dim"]
            mean = s.sum(-1, keepdim=True) / n
            variance = ((s - mean) ** 2).sum(-1, keepdim=True) / n
            h = (s - mean) / torch.sqrt(variance + EPS) * wide["w"] + wide["b"]
            r["h"] = h.detach()
            heads, grads = heads + [h], grads + ([state["dh"].double()] if train else [])
        if train:
            names = [k for k in ("z", "y", "w", "b") if k in wide]
            for k, d in zip(names, torch.autograd.grad(heads, [wide[k] for k in names], grads)):
                r["d" + k] = d
    return r
