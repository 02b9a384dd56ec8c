"""Cases of the MLP layer's operators: the product with its epilogue, its two gradient products, the epilogue's
gradient, and dropout.

    linear     Y[N,M] = R + D(act(X[N,K] W[K,M] + b)),  Z = X W + b kept for the backward pass where asked for
    dx         dX[N,K] = R + dZ[N,M] W[K,M]^T
    dw         dW[K,M] = R + X[N,K]^T dZ[N,M]
    act_grad   dZ = D(dY) act'(Z),  dbias = the column sums of dZ before it is rounded
    dropout    Y = R + D(X)

D drops an element where a 16-bit number of a counter-based generator is below t = rint(65536 p) and multiplies the
others by 65536 / (65536 - t).  The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
numbers: as easy as 1, 2, 3", 2011): key = the seed's two words, counter = (column / 8, row, the offset's two words);
column c takes half-word c % 8 of the 128 bits, low halves first.
"""
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
LARGEST = 2048 * 4096 * 11008


def listed():
    return [
        # one token through the up projection of a served MLP: the weights' bytes are the cost
        {"name": "linear decode 1", "op": "linear", "type": "bf16", "N": 1, "K": 4096, "M": 11008, "act": "silu",
         "bias": True, "residual": False, "preact": False, "p": 0.0},
        # a batch of decoding sequences through the down projection, into the residual stream
        {"name": "linear decode 13", "op": "linear", "type": "f16", "N": 13, "K": 11008, "M": 4096, "act": "none",
         "bias": True, "residual": True, "preact": False, "p": 0.0},
        # a short ragged prompt on a small model, trained with dropout: latency
        {"name": "linear ragged", "op": "linear", "type": "f16", "N": 77, "K": 1000, "M": 1336, "act": "gelu",
         "bias": True, "residual": True, "preact": True, "p": 0.1},
        # a training step's up projection
        {"name": "linear train", "op": "linear", "type": "bf16", "N": 2048, "K": 4096, "M": 11008, "act": "gelu_tanh",
         "bias": True, "residual": False, "preact": True, "p": 0.0},
        # its gradient with respect to the layer's input, added to the residual path's gradient
        {"name": "dx train", "op": "dx", "type": "bf16", "N": 2048, "K": 4096, "M": 11008, "residual": True},
        # the same for a short ragged batch
        {"name": "dx ragged", "op": "dx", "type": "f16", "N": 200, "K": 1000, "M": 4096, "residual": False},
        # the weights' gradient of a training step
        {"name": "dw train", "op": "dw", "type": "bf16", "out": "bf16", "N": 2048, "K": 4096, "M": 11008,
         "residual": False},
        # a small layer's, added to what earlier micro-batches left in 32 bits
        {"name": "dw accumulate", "op": "dw", "type": "f16", "out": "f32", "N": 333, "K": 1032, "M": 2056,
         "residual": True},
        # the epilogue's gradient of a training step, dropout behind the activation
        {"name": "act_grad train", "op": "act_grad", "type": "bf16", "N": 2048, "M": 11008, "act": "gelu", "p": 0.1},
        # of a few rows of odd length
        {"name": "act_grad ragged", "op": "act_grad", "type": "f16", "N": 37, "M": 1003, "act": "silu", "p": 0.0},
        # dropout of a training step's hidden states into the residual stream
        {"name": "dropout train", "op": "dropout", "type": "bf16", "N": 4096, "M": 4096, "p": 0.1, "residual": True},
        # of a few rows: latency
        {"name": "dropout ragged", "op": "dropout", "type": "f16", "N": 33, "M": 4104, "p": 0.5, "residual": False},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, uniform over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def _width(rng, lo, hi):
    """A row length: mostly a multiple of 8, as layers have it, sometimes any number."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "dx", "dw", "act_grad", "dropout"])
    c = {"op": op, "type": rng.choice(["f16", "bf16"])}
    if op in ("linear", "dx", "dw"):
        while True:
            n, k, m = _spread(rng, 1, 4096), _width(rng, 64, 11008), _width(rng, 64, 11008)
            if n * k * m <= LARGEST and k * m <= 4096 * 11008:
                break
        c.update(N=n, K=k, M=m, residual=rng.random() < 0.5)
        if op == "linear":
            c.update(act=rng.choice(list(ACTS)), bias=rng.random() < 0.7, preact=rng.random() < 0.4,
                     p=rng.choice([0.0, 0.0, round(rng.uniform(0.02, 0.5), 3)]))
        if op == "dw":
            c.update(out=rng.choice([c["type"], "f32"]))
        return c
    while True:
        n, m = _spread(rng, 1, 16384), _width(rng, 64, 11008)
        if n * m <= 2048 * 11008:
            break
    c.update(N=n, M=m, p=round(rng.uniform(0.02, 0.5), 3))
    if op == "act_grad":
        c.update(act=rng.choice(list(ACTS)))
        if rng.random() < 0.3:
            c.update(p=0.0)
    else:
        c.update(residual=rng.random() < 0.5)
    return c


def _operands(case, seed):
    """The inputs alone: activations of unit size, weights that keep it, gradients a good deal smaller."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    op, n, m, k = case["op"], case["N"], case["M"], case.get("K", 0)
    s = {"seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) & (2**64 - 1), "offset": (seed << 20) + 7}
    if op == "linear":
        s.update(x=normal(n, k), w=normal(k, m, scale=k**-0.5))
        if case["bias"]:
            s["b"] = normal(m, scale=0.1)
        if case["residual"]:
            s["r"] = normal(n, m)
    elif op == "dx":
        s.update(dz=normal(n, m, scale=0.05), w=normal(k, m, scale=k**-0.5))
        if case["residual"]:
            s["r"] = normal(n, k, scale=0.05)
    elif op == "dw":
        s.update(x=normal(n, k), dz=normal(n, m, scale=0.05))
        if case["residual"]:
            s["r"] = normal(k, m, scale=0.05 * n**0.5, dtype=TYPES[case["out"]])
    elif op == "act_grad":
        s.update(dy=normal(n, m, scale=0.05))
        if case["act"] != "none":
            s["z"] = normal(n, m)
    else:
        s.update(x=normal(n, m))
        if case["residual"]:
            s["r"] = normal(n, m)
    return s


def prepare(case, seed):
    s = _operands(case, seed)
    s["case"] = case
    t = TYPES[case["type"]]
    n, m, k = case["N"], case["M"], case.get("K", 0)
    op = case["op"]

    def out(rows, cols, dtype=t):
        return torch.empty(rows, cols, dtype=dtype, device="cuda")

    # the buffers that a program keeps for the results
    if op == "linear":
        s["y"] = out(n, m)
        if case["preact"]:
            s["z"] = out(n, m)
    elif op == "dx":
        s["dx"] = out(n, k)
    elif op == "dw":
        s["dw"] = out(k, m, TYPES[case["out"]])
    elif op == "act_grad":
        s["dz"], s["dbias"] = out(n, m), torch.empty(m, dtype=torch.float32, device="cuda")
    else:
        s["y"] = out(n, m)
    return s


# ---- the framework's calls -----------------------------------------------------------------

_G = None


def _framework():
    global _G
    if _G is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "fp8-mlp-metal41-bench_b200"))
        from mlpgemm import lib
        lib.init(torch.cuda.current_device())
        _G = lib
    return _G


def _workspace(s, G, op, a, b, case):
    """The workspace that the call needs, kept with the state (None for most shapes)."""
    if "ws" not in s:
        size = G.linear_workspace(op, a, b, case["N"], case["K"], case["M"])
        s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
        s["wsb"] = size
    return s["ws"], s["wsb"]


def _run_own(s):
    G, case = _framework(), s["case"]
    op, n, m = case["op"], case["N"], case["M"]
    dev, st = s_device(), torch.cuda.current_stream().cuda_stream
    ty = G.TYPES[case["type"]]
    if op == "linear":
        ws, wsb = _workspace(s, G, G.OP_LINEAR, s["x"], s["w"], case)
        G.linear(dev, ty, s["x"], s["w"], s["y"], n, case["K"], m, bias=s.get("b"), act=ACTS[case["act"]],
                 residual=s.get("r"), preact=s.get("z"), dropout_p=case["p"], seed=s["seed"], offset=s["offset"],
                 workspace=ws, workspace_bytes=wsb, stream=st)
        return {"y": s["y"], "z": s["z"]} if case["preact"] else {"y": s["y"]}
    if op == "dx":
        ws, wsb = _workspace(s, G, G.OP_DX, s["dz"], s["w"], case)
        G.linear_dx(dev, ty, s["dz"], s["w"], s["dx"], n, case["K"], m, residual=s.get("r"), workspace=ws,
                    workspace_bytes=wsb, stream=st)
        return {"dx": s["dx"]}
    if op == "dw":
        ws, wsb = _workspace(s, G, G.OP_DW, s["x"], s["dz"], case)
        G.linear_dw(dev, ty, s["x"], s["dz"], s["dw"], n, case["K"], m, out_type=G.TYPES[case["out"]],
                    residual=s.get("r"), workspace=ws, workspace_bytes=wsb, stream=st)
        return {"dw": s["dw"]}
    if op == "act_grad":
        G.act_grad(dev, ty, s["dy"], s.get("z"), s["dz"], s["dbias"], n, m, act=ACTS[case["act"]],
                   dropout_p=case["p"], seed=s["seed"], offset=s["offset"], stream=st)
        return {"dz": s["dz"], "dbias": s["dbias"]}
    G.dropout(dev, ty, s["x"], s["y"], n, m, case["p"], s["seed"], s["offset"], residual=s.get("r"), stream=st)
    return {"y": s["y"]}


def s_device():
    return torch.cuda.current_device()


# ---- the plain forms ------------------------------------------------------------------------

_LOW = 0xFFFFFFFF


def _numbers(rows, cols, seed, offset):
    """The generator's 16-bit numbers [rows, cols]; products of two 32-bit words wrap in the 64 bits as they should."""
    groups = (cols + 7) // 8
    c0 = torch.arange(groups, device="cuda")[None, :].expand(rows, groups)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, groups)
    c2 = torch.full_like(c0, offset & _LOW)
    c3 = torch.full_like(c0, offset >> 32)
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, groups * 8)[:, :cols]


def _dropped(v, case, s):
    t = round(case["p"] * 65536)
    if t == 0:
        return v
    keep = _numbers(v.shape[0], v.shape[1], s["seed"], s["offset"]) >= t
    return torch.where(keep, v * (65536 / (65536 - t)), 0.0)


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5**0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5**0.5)) + z * torch.exp(-0.5 * z * z) * (2 * np.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / np.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    op, t = case["op"], TYPES[case["type"]]
    r = s["r"].float() if "r" in s else None
    if op == "linear":
        z = s["x"].float() @ s["w"].float()
        if "b" in s:
            z = z + s["b"].float()
        y = _dropped(_act(z, case["act"]), case, s)
        y = (y if r is None else r + y).to(t)
        return {"y": y, "z": z.to(t)} if case["preact"] else {"y": y}
    if op == "dx":
        v = s["dz"].float() @ s["w"].float().t()
        return {"dx": (v if r is None else r + v).to(t)}
    if op == "dw":
        v = s["x"].float().t() @ s["dz"].float()
        return {"dw": (v if r is None else r + v).to(TYPES[case["out"]])}
    if op == "act_grad":
        v = _dropped(s["dy"].float(), case, s)
        if case["act"] != "none":
            v = v * _slope(s["z"].float(), case["act"])
        return {"dz": v.to(t), "dbias": v.sum(0)}
    v = _dropped(s["x"].float(), case, s)
    return {"y": (v if r is None else r + v).to(t)}


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    e, n, m, k = 2, case["N"], case["M"], case.get("K", 0)
    op = case["op"]
    if op == "linear":
        size = n * k + k * m + n * m + (m if case["bias"] else 0)
        size += (n * m if case["residual"] else 0) + (n * m if case["preact"] else 0)
        return {"bytes": e * size, "flops": 2 * n * k * m}
    if op == "dx":
        return {"bytes": e * (n * m + k * m + n * k * (2 if case["residual"] else 1)), "flops": 2 * n * k * m}
    if op == "dw":
        o = 4 if case["out"] == "f32" else 2
        return {"bytes": e * (n * k + n * m) + o * k * m * (2 if case["residual"] else 1), "flops": 2 * n * k * m}
    if op == "act_grad":
        return {"bytes": e * n * m * (2 if case["act"] == "none" else 3) + 4 * m, "flops": 12 * n * m}
    return {"bytes": e * n * m * (3 if case["residual"] else 2), "flops": 4 * n * m}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _keep64(rows, cols, p, seed, offset):
    """D's factor for every element, from the generator's definition in numpy's unsigned integers."""
    t = int(np.rint(p * 65536))
    groups = -(-cols // 8)
    ctr = np.zeros((4, rows, groups), np.uint64)
    ctr[0] = np.arange(groups, dtype=np.uint64)
    ctr[1] = np.arange(rows, dtype=np.uint64)[:, None]
    ctr[2], ctr[3] = offset % 2**32, offset // 2**32
    key = [seed % 2**32, seed // 2**32]
    mult, weyl = (np.uint64(0xD2511F53), np.uint64(0xCD9E8D57)), (0x9E3779B9, 0xBB67AE85)
    low, half = np.uint64(2**32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = ctr[0] * mult[0], ctr[2] * mult[1]
        ctr = np.stack([(b >> half) ^ ctr[1] ^ np.uint64(key[0]), b & low,
                        (a >> half) ^ ctr[3] ^ np.uint64(key[1]), a & low])
        key = [(key[i] + weyl[i]) % 2**32 for i in range(2)]
    number = np.empty((rows, groups, 8), np.uint16)
    for i in range(8):
        number[:, :, i] = (ctr[i // 2] >> np.uint64(16 * (i % 2))) & np.uint64(0xFFFF)
    number = number.reshape(rows, groups * 8)[:, :cols]
    return torch.from_numpy(np.where(number >= t, 65536.0 / (65536 - t), 0.0)).cuda()


def _normal_cdf(z):
    return 0.5 * torch.special.erfc(-z / 2**0.5)


def _act64(z, act):
    if act == "gelu_tanh":
        return z * torch.sigmoid((8 / np.pi) ** 0.5 * (z + 0.044715 * z**3))
    return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "gelu": lambda: z * _normal_cdf(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def _slope64(z, act):
    if act == "relu":
        return torch.where(z > 0, 1.0, 0.0).double()
    if act == "gelu":
        return _normal_cdf(z) + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5
    if act == "gelu_tanh":
        c = (8 / np.pi) ** 0.5
        q = torch.sigmoid(c * (z + 0.044715 * z**3))
        return q + z * q * (1 - q) * c * (1 + 0.134145 * z**2)
    q = torch.sigmoid(z)
    return q + z * q * (1 - q)


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) else v for k, v in _operands(case, seed).items()}
    op = case["op"]
    d = 1.0
    if case.get("p", 0.0) > 0:
        d = _keep64(case["N"], case["M"], case["p"], s["seed"], s["offset"])
    r = s.get("r", 0.0)
    if op == "linear":
        z = torch.mm(s["x"], s["w"]) + s.get("b", 0.0)
        y = r + d * _act64(z, case["act"])
        return {"y": y, "z": z} if case["preact"] else {"y": y}
    if op == "dx":
        return {"dx": r + torch.mm(s["dz"], s["w"].t())}
    if op == "dw":
        return {"dw": r + torch.mm(s["x"].t(), s["dz"])}
    if op == "act_grad":
        v = d * s["dy"]
        if case["act"] != "none":
            v = v * _slope64(s["z"], case["act"])
        return {"dz": v, "dbias": v.sum(0)}
    return {"y": r + d * s["x"]}
