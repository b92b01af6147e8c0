"""Cases of the operators on weights held in four bits: making such a matrix, the product with one, and the gated pair of products
that opens a feed-forward.  `run` takes a case through the framework where `own` is true, and through elementary torch operations
where it is not.

A row of a matrix is cut into groups of 32, 64 or 128 neighbours.  A group keeps a bfloat16 scale s and offset b, its elements a
code q of four bits each, and stands for W = bfloat16(q s + b).  Codes lie as int32 [rows / 16, K / 64, 4, 8, 2, 2]: row
16 i + 8 h + r, k = 64 c + 16 t + 8 w + 2 p + e is bits 4 (4 e + p) of [i, c, t, r, h, w]; scales and offsets as bfloat16
[rows / 16, groups, 8, 2, 2] with the row as above and (s, b) last.  Rows and groups beyond the matrix are zeros.
"""
import math

import torch

own = False

LARGEST = 2 * 2048 * 2 * 12288 * 4096      # operations of the largest product listed
MOST_WEIGHTS = 151936 * 2560               # and the most weights


def listed():
    return [
        # the output projection of a small model for one request: little to read, the call itself counts
        dict(name="product_1_small", op="product", rows=1, n=2048, k=2048, group=64, bias=False, out="bfloat16"),
        # ... and of a middle-sized one, groups of 128
        dict(name="product_1", op="product", rows=1, n=4096, k=4096, group=128, bias=False, out="bfloat16"),
        # the fused query, key and value projection, with a bias, of eight decoding requests
        dict(name="product_8", op="product", rows=8, n=7168, k=5120, group=64, bias=True, out="bfloat16"),
        # the output head over a large vocabulary: float32 logits of four requests
        dict(name="head_4", op="product", rows=4, n=151936, k=2560, group=64, bias=False, out="float32"),
        # odd sizes: rows that fill no tile, a depth that ends inside one, small groups
        dict(name="product_ragged", op="product", rows=37, n=1003, k=1056, group=32, bias=True, out="float32"),
        # the way down of a feed-forward for a prompt of 2,048 tokens
        dict(name="product_prompt", op="product", rows=2048, n=4096, k=12288, group=64, bias=False, out="bfloat16"),
        # the gated pair: one request, a batch of eight, a step that mixes requests and a short prompt, a whole prompt
        dict(name="gated_1", op="gated", rows=1, n=12288, k=4096, group=64, activation="silu"),
        dict(name="gated_8", op="gated", rows=8, n=17408, k=5120, group=64, activation="silu"),
        dict(name="gated_77", op="gated", rows=77, n=9728, k=2560, group=128, activation="gelu_pytorch_tanh"),
        dict(name="gated_prompt", op="gated", rows=2048, n=12288, k=4096, group=128, activation="silu"),
        # loading: a small projection, a large one
        dict(name="quantise_small", op="quantise", n=1000, k=2080, group=32, stored="float32"),
        dict(name="quantise", op="quantise", n=12288, k=4096, group=64, stored="bfloat16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["product", "product", "gated", "gated", "quantise"])
    group = rng.choice([32, 64, 128])
    n = _spread(rng, 16, 20000)
    k = group * max(1, round(_spread(rng, 64, 18000) / group))
    if op == "quantise":
        k = min(k, max(group, MOST_WEIGHTS // 4 // n // group * group))
        return dict(op=op, n=n, k=k, group=group, stored=rng.choice(["bfloat16", "float32"]))
    rows = _spread(rng, 1, 2048)
    rows = max(1, min(rows, LARGEST // (n * k * (4 if op == "gated" else 2))))
    if op == "gated":
        return dict(op=op, rows=rows, n=n, k=k, group=group, activation=rng.choice(["silu", "gelu", "gelu_pytorch_tanh", "relu"]))
    return dict(op=op, rows=rows, n=n, k=k, group=group, bias=rng.random() < 0.5, out=rng.choice(["bfloat16", "float32"]))


# ---- the format, in torch ----
def _quantise(w, group):
    """Codes [N, K] (int32), scales and offsets [N, K / group] (bfloat16) of a float32 matrix."""
    n, k = w.shape
    parts = w.view(n, k // group, group)
    low, high = parts.amin(2), parts.amax(2)
    fifteen = torch.full((1, 1), 15, dtype=w.dtype, device=w.device)   # (a number instead would be multiplied by as 1 / 15)
    scale, offset = ((high - low) / fifteen).to(torch.bfloat16), low.to(torch.bfloat16)
    s, b = scale.float()[:, :, None], offset.float()[:, :, None]
    q = torch.where(s > 0, (parts - b) / s, torch.zeros_like(parts)).round_().clamp_(0, 15)
    return q.view(n, k).to(torch.int32), scale, offset


def _pack(q, scale, offset, group):
    n, k = q.shape
    tiles, blocks = -(-n // 16), -(-k // 64)
    full = torch.zeros(tiles * 16, blocks * 64, dtype=torch.int32, device=q.device)
    full[:n, :k] = q
    full = full.view(tiles, 2, 8, blocks, 4, 2, 4, 2).permute(0, 3, 4, 2, 1, 5, 7, 6)   # [i, c, t, r, h, w, e, p]
    codes = torch.zeros(full.shape[:6], dtype=torch.int32, device=q.device)
    for e in range(2):
        for p in range(4):
            codes |= full[..., e, p] << (4 * (4 * e + p))
    groups = max(1, blocks * 64 // group)
    affine = torch.zeros(tiles * 16, groups, 2, dtype=torch.bfloat16, device=q.device)
    affine[:n, :k // group, 0] = scale
    affine[:n, :k // group, 1] = offset
    return codes, affine.view(tiles, 2, 8, groups, 2).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(codes, affine, n, k, group):
    """The float32 matrix that codes, scales and offsets stand for, every element a bfloat16 value."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=codes.device).view(2, 4)
    q = (codes[..., None, None] >> shifts) & 15
    q = q.permute(0, 4, 3, 1, 2, 5, 7, 6).reshape(codes.shape[0] * 16, -1)[:n, :k]
    a = affine.permute(0, 3, 2, 1, 4).reshape(codes.shape[0] * 16, -1, 2)[:n, :k // group].float()
    w = q.view(n, k // group, group) * a[:, :, :1] + a[:, :, 1:]
    return w.to(torch.bfloat16).float().view(n, k)


def _activation(z, name):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_pytorch_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return torch.where(z > 0, z, torch.zeros_like(z))


# ---- the cases ----
def _weights(case, g):
    """Normal weights whose rows differ in size, as trained ones do."""
    n, k = case["n"], case["k"]
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    return w.mul_(0.5 + torch.rand(n, 1, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, k, group = case["n"], case["k"], case["group"]
    state = dict(case=case)
    if case["op"] == "quantise":
        state["w"] = _weights(case, g).to(getattr(torch, case["stored"]))
        return state
    x = torch.randn(case["rows"], k, generator=g, device="cuda")
    x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 8   # (a few channels of a normed stream are large)
    state["x"] = x.to(torch.bfloat16)
    state["packed"] = [_pack(*_quantise(_weights(case, g), group), group) for _ in range(2 if case["op"] == "gated" else 1)]
    if case.get("bias"):
        state["bias"] = torch.randn(n, generator=g, device="cuda") * 0.1
    if own:   # the handles that a model keeps of the same tensors
        from velox_b200.csrc import ops
        state["matrices"] = [ops.Q4Matrix(codes, affine, n, k, group) for codes, affine in state["packed"]]
    return state


def run(state):
    case = state["case"]
    n, k, group = case["n"], case["k"], case["group"]
    if own:
        from velox_b200.csrc import ops
        if case["op"] == "quantise":
            return ops.dequantize_q4(ops.quantize_q4(state["w"], group))
        if case["op"] == "gated":
            return ops.gated_q4(state["x"], state["matrices"][0], state["matrices"][1], case["activation"], w_ready=True)
        return ops.gemm_q4(state["x"], state["matrices"][0], state.get("bias"), getattr(torch, case["out"]), w_ready=True)
    if case["op"] == "quantise":
        q, scale, offset = _quantise(state["w"].float(), group)
        return _unpack(*_pack(q, scale, offset, group), n, k, group).to(torch.bfloat16)
    x = state["x"].float()
    sums = [x @ _unpack(codes, affine, n, k, group).t() for codes, affine in state["packed"]]
    if case["op"] == "gated":
        return (_activation(sums[0], case["activation"]) * sums[1]).to(torch.bfloat16)
    if case["bias"]:
        sums[0] = sums[0] + state["bias"]
    return sums[0].to(getattr(torch, case["out"]))


def work(case):
    n, k, group = case["n"], case["k"], case["group"]
    if case["op"] == "quantise":   # the stored matrix in, the matrix that the codes stand for out
        return {"bytes": n * k * ((2 if case["stored"] == "bfloat16" else 4) + 2), "flops": 0}
    rows, matrices = case["rows"], 2 if case["op"] == "gated" else 1
    weights = matrices * (n * k / 2 + 4 * n * k / group)
    out = rows * n * (4 if case.get("out") == "float32" else 2)
    return {"bytes": weights + 2 * rows * k + out + (4 * n if case.get("bias") else 0), "flops": 2 * matrices * rows * n * k}


# ---- the operators' definition in 64 bits ----
def _matrix64(codes, affine, n, k, group):
    """[n, k] in 64 bits: each element looked up by its own row and column."""
    rows, cols = torch.arange(n, device="cuda")[:, None], torch.arange(k, device="cuda")[None, :]
    i, h, r = rows // 16, rows // 8 % 2, rows % 8
    c, t, w, p, e = cols // 64, cols // 16 % 4, cols // 8 % 2, cols // 2 % 4, cols % 2
    shape = codes.shape
    at = ((((i * shape[1] + c) * 4 + t) * 8 + r) * 2 + h) * 2 + w
    q = (codes.reshape(-1)[at].to(torch.int64) >> (16 * e + 4 * p)) & 15
    del at
    place = ((i * affine.shape[1] + cols // group) * 8 + r) * 2 + h
    pairs = affine.reshape(-1, 2)
    value = q.double() * pairs[:, 0].double()[place] + pairs[:, 1].double()[place]
    return value.to(torch.bfloat16).double()


def exact(case, seed):
    state = prepare(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    if case["op"] == "quantise":
        w = state["w"].double()
        out, steps = torch.empty_like(w), torch.full((n, 1), 15, dtype=torch.float64, device="cuda")
        for at in range(0, k, group):
            part = w[:, at:at + group]
            low, high = part.min(1, keepdim=True).values, part.max(1, keepdim=True).values
            s, b = ((high - low) / steps).to(torch.bfloat16).double(), low.to(torch.bfloat16).double()
            q = torch.nan_to_num((part - b) / s, nan=0.0).round().clamp(0, 15)
            out[:, at:at + group] = (q * s + b).to(torch.bfloat16).double()
        return out
    x, sums = state["x"].double(), []
    step = max(1, (1 << 26) // k // 16) * 16   # rows of the matrix at a time
    for codes, affine in state["packed"]:
        parts = [x @ _matrix64(codes[at // 16:], affine[at // 16:], min(step, n - at), k, group).t() for at in range(0, n, step)]
        sums.append(torch.cat(parts, 1))
    if case["op"] == "product":
        return sums[0] + (state["bias"].double() if case["bias"] else 0)
    gate = sums[0]
    if case["activation"] == "silu":
        gate = gate * torch.special.expit(gate)
    elif case["activation"] == "gelu":
        gate = gate * torch.special.ndtr(gate)
    elif case["activation"] == "gelu_pytorch_tanh":
        gate = gate * torch.special.expit(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))
    else:
        gate = gate.clamp(min=0)
    return gate * sums[1]
