"""The grouped and the 8-bit matrix products on fixed cases: the library's calls beside plain torch operations.

A case is one call as a program makes it.  `op` says which:

  product   C_g = op(A_g) B_g for the columns of every group (an expert's tokens, a window's columns)
  outer     D_g = X_g Y_g^T (+ D_g), the gradient of the group's matrix
  int8      y = (W q) scaled, q the columns of x rounded to 8 bits with one scale a column; W 8 bits, one scale a channel

The matrices of the library are column-major; a tensor of shape (columns, rows) is such a matrix, so a token
is a column and a weight tensor (out, in) is A with op(A) = A^T.  Groups are ragged: every token picks `top_k` of the
`groups` at random with some of them preferred, and the columns of a group lie side by side.
"""
import functools
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


def listed():
    return [
        # one token through its experts while text is generated: eight columns, each with a matrix of its own
        {"name": "product one token", "op": "product", "type": "bf16", "trans": "T", "tokens": 1, "top_k": 8, "groups": 64, "m": 1024, "k": 2048, "pad": 0},
        # a batch of 64 running sequences: nearly every expert is met, by a few columns each
        {"name": "product decode batch", "op": "product", "type": "bf16", "trans": "T", "tokens": 64, "top_k": 4, "groups": 32, "m": 2048, "k": 1408, "pad": 0},
        # the gradient of the inputs of a mid-sized layer whose sizes are multiples of nothing
        {"name": "product inputs' gradient odd", "op": "product", "type": "f16", "trans": "N", "tokens": 1501, "top_k": 2, "groups": 16, "m": 1001, "k": 1433, "pad": 3},
        # a training step's forward product, the largest
        {"name": "product large", "op": "product", "type": "bf16", "trans": "T", "tokens": 16384, "top_k": 2, "groups": 16, "m": 4096, "k": 2048, "pad": 0},
        # window transformations applied from the left to what is right of each window, in the library's own precision
        {"name": "product f64 windows", "op": "product", "type": "f64", "trans": "T", "tokens": 40000, "top_k": 1, "groups": 24, "m": 312, "k": 312, "pad": 0},
        # gradients of the matrices of a large layer, held in 32 bits
        {"name": "outer large", "op": "outer", "type": "bf16", "out": "f32", "beta": 0.0, "tokens": 16384, "top_k": 2, "groups": 16, "m": 2048, "n": 4096, "pad": 0},
        # a small odd layer of many groups, some with hardly a column, the gradients in the operands' type
        {"name": "outer odd", "op": "outer", "type": "f16", "out": "f16", "beta": 0.0, "tokens": 1388, "top_k": 2, "groups": 24, "m": 721, "n": 1337, "pad": 1},
        # one matrix for all columns, a small projection over a long batch: added to what earlier micro-batches left
        {"name": "outer one group", "op": "outer", "type": "bf16", "out": "f32", "beta": 1.0, "tokens": 20000, "top_k": 1, "groups": 1, "m": 512, "n": 384, "pad": 0},
        # one token through a projection
        {"name": "int8 one token", "op": "int8", "type": "bf16", "tokens": 1, "top_k": 1, "groups": 1, "m": 4096, "k": 4096, "pad": 0},
        # a small odd prompt
        {"name": "int8 odd", "op": "int8", "type": "f16", "tokens": 333, "top_k": 1, "groups": 1, "m": 1999, "k": 1403, "pad": 0},
        # experts over a batch
        {"name": "int8 experts", "op": "int8", "type": "f16", "tokens": 3000, "top_k": 2, "groups": 32, "m": 1536, "k": 2048, "pad": 0},
        # a long prompt through a projection
        {"name": "int8 large", "op": "int8", "type": "bf16", "tokens": 8192, "top_k": 1, "groups": 1, "m": 8192, "k": 4096, "pad": 0},
    ]


def draw(rng):
    def size(low, high):
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return max(low, v // 64 * 64 if rng.random() < 0.5 else v)

    op = rng.choice(["product", "product", "outer", "int8"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16"] if op == "int8" else ["bf16", "bf16", "f16", "f16", "f64"])}
    case["groups"] = rng.choice([1, size(2, 64)])
    case["top_k"] = min(case["groups"], rng.choice([1, 2, 4, 8]))
    case["m"] = size(64, 4096)
    case["n" if op == "outer" else "k"] = inner = size(64, 4096)
    while case["groups"] * case["m"] * inner > 1 << 28:         # the matrices' room: at most that of 16 of the largest
        case["groups"] = case["groups"] // 2
        case["top_k"] = min(case["groups"], case["top_k"])
    most = 1e10 if case["type"] == "f64" else 2.5e11            # multiply-adds
    most = int(most / (case["m"] * inner * case["top_k"]))
    case["tokens"] = max(1, min(size(1, 16384), most))
    if op == "product":
        case["trans"] = rng.choice(["T", "N"])
    if op == "outer":
        case["out"] = rng.choice([case["type"], "f64" if case["type"] == "f64" else "f32"])
        case["beta"] = rng.choice([0.0, 1.0])
    case["pad"] = rng.choice([0, 0, 0, 1, 8])
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    groups, columns = case["groups"], case["tokens"] * case["top_k"]

    def matrix(*shape, scale=1.0, dtype=kind):
        full = torch.empty(*shape[:-1], shape[-1] + case["pad"], device="cuda", dtype=dtype)
        full.normal_(generator=gen).mul_(scale)
        return full[..., : shape[-1]]

    # the router's choice: the top_k largest of the groups' scores, and the columns in the groups' order
    score = torch.randn(groups, generator=gen, device="cuda") * 0.5
    score = score - torch.log(torch.rand(case["tokens"], groups, generator=gen, device="cuda").clamp_min(1e-20).log().neg())
    chosen = score.topk(case["top_k"], dim=1).indices.reshape(-1)
    counts = torch.bincount(chosen, minlength=groups)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    state = {"case": case, "offsets": offsets, "sizes": counts.tolist()}
    m = case["m"]
    if case["op"] == "product":
        k = case["k"]
        shape = (groups, m, k) if case["trans"] == "T" else (groups, k, m)
        state |= {"A": matrix(*shape, scale=k ** -0.5), "B": matrix(columns, k)}
    elif case["op"] == "outer":
        n = case["n"]
        state |= {"X": matrix(columns, m), "Y": matrix(columns, n, scale=0.1)}
        if case["beta"]:
            state["D"] = matrix(groups, n, m, dtype=TYPES[case["out"]])
    else:
        k = case["k"]
        x = matrix(columns, k)
        x[:, torch.randint(0, k, (max(1, k // 100),), generator=gen, device="cuda")] *= 8       # the channels that stand out
        weight = torch.randint(-127, 128, (groups, m, k + case["pad"]), generator=gen, device="cuda", dtype=torch.int8)[..., :k]
        state |= {"x": x, "W": weight, "scale": torch.rand(groups, m, generator=gen, device="cuda") * (0.02 * k ** -0.5) + 1e-4 * k ** -0.5}
    return state


@functools.lru_cache(maxsize=None)
def _library():
    import starneig_amd as S
    if not S.node_initialized():
        S.node_init(1, 1, S.NO_MESSAGES)
    return S


def _own(state):
    S, case = _library(), state["case"]
    if case["op"] == "product":
        A, B = state["A"], state["B"]
        C = torch.empty(B.shape[0], case["m"], device=B.device, dtype=B.dtype)
        rc = S.grouped_gemm_device(case["trans"], state["offsets"], A, B, C)
    elif case["op"] == "outer":
        X, Y = state["X"], state["Y"]
        # the sum over micro-batches is kept apart from the state here, so that a pass can be called again
        C = state["D"].clone() if case["beta"] else torch.empty(case["groups"], case["n"], case["m"], device=X.device, dtype=TYPES[case["out"]])
        rc = S.grouped_outer_device(state["offsets"], X, Y, C, beta=case["beta"])
    else:
        x, W = state["x"], state["W"]
        q = torch.empty(x.shape, device=x.device, dtype=torch.int8)
        scale = torch.empty(x.shape[0], device=x.device)
        C = torch.empty(x.shape[0], case["m"], device=x.device, dtype=x.dtype)
        rc = S.quantize_i8_device(x, q, scale)
        if rc == 0 and case["groups"] == 1:
            rc = S.gemm_i8_device(W[0], state["scale"][0], q, scale, C)
        elif rc == 0:
            rc = S.grouped_gemm_i8_device(state["offsets"], W, state["scale"], q, scale, C)
    if rc != 0:
        raise RuntimeError("the library returned %d" % rc)
    return C


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _whole_product(q, w):
    """q w^T of whole numbers up to 127: sums of 1024 products fit 24 bits, so each chunk is exact in 32-bit floats."""
    parts = [a @ b.t() for a, b in zip(q.split(1024, 1), w.float().split(1024, 1))]
    return parts[0] if len(parts) == 1 else sum(p.double() for p in parts).float()


def run(state):
    if own:
        return _own(state)
    case, sizes = state["case"], state["sizes"]
    if case["op"] == "product":
        some = [g for g, s in enumerate(sizes) if s]
        parts = state["B"].split([s for s in sizes if s])
        if case["trans"] == "T":
            C = [_wide(b) @ _wide(state["A"][g]).t() for g, b in zip(some, parts)]
        else:
            C = [_wide(b) @ _wide(state["A"][g]) for g, b in zip(some, parts)]
        return torch.cat(C).to(state["B"].dtype)
    if case["op"] == "outer":
        D = torch.stack([_wide(y).t() @ _wide(x) for x, y in zip(state["X"].split(sizes), state["Y"].split(sizes))])
        if case["beta"]:
            D = D + case["beta"] * _wide(state["D"])
        return D.to(TYPES[case["out"]])
    x = state["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    q = torch.where(scale > 0, x / scale, torch.zeros_like(x)).round()
    some = [g for g, s in enumerate(sizes) if s]
    y = torch.cat([_whole_product(b, state["W"][g]) * state["scale"][g] for g, b in zip(some, q.split([s for s in sizes if s]))])
    return (y * scale).to(state["x"].dtype)


def exact(case, seed):
    state = prepare(case, seed)
    ends = torch.tensor(state["sizes"]).cumsum(0).tolist()
    spans = list(zip([0] + ends[:-1], ends))
    wide = torch.float64
    if case["op"] == "product":
        C = torch.empty(ends[-1], case["m"], device="cuda", dtype=wide)
        for g, (a, b) in enumerate(spans):
            W = state["A"][g].to(wide)
            C[a:b] = torch.matmul(state["B"][a:b].to(wide), W.transpose(0, 1) if case["trans"] == "T" else W)
        return C
    if case["op"] == "outer":
        D = torch.zeros(case["groups"], case["n"], case["m"], device="cuda", dtype=wide)
        for g, (a, b) in enumerate(spans):
            D[g] = torch.matmul(state["Y"][a:b].to(wide).transpose(0, 1), state["X"][a:b].to(wide))
        return D + case["beta"] * state["D"].to(wide) if case["beta"] else D
    C = torch.empty(ends[-1], case["m"], device="cuda", dtype=wide)
    for g, (a, b) in enumerate(spans):
        x = state["x"][a:b].to(wide)
        # the scale is a 32-bit number by definition
        scale = (x.abs().max(dim=1, keepdim=True).values / 127).float().to(wide) if b > a else x[:, :1]
        q = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale)))
        C[a:b] = torch.matmul(q, state["W"][g].to(wide).transpose(0, 1)) * state["scale"][g].to(wide) * scale
    return C


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}
    columns, groups, m = case["tokens"] * case["top_k"], case["groups"], case["m"]
    inner = case["n"] if case["op"] == "outer" else case["k"]
    met = groups * (1 - (1 - case["top_k"] / groups) ** case["tokens"])         # groups with a column, as even choices have them
    one = size[case["type"]]
    if case["op"] == "outer":
        nbytes = columns * (m + inner) * one + groups * m * inner * size[case["out"]] * (2 if case["beta"] else 1)
    elif case["op"] == "product":
        nbytes = columns * (m + inner) * one + met * m * inner * one
    else:
        nbytes = columns * (m + inner) * one + met * (m * inner + 4 * m)
    return {"bytes": nbytes, "flops": 2.0 * columns * m * inner}
