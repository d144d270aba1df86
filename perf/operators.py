"""The row operators between the matrix products of a decoder: layer norm, rotary positions, routing to experts and
token log-probabilities, as cases to time and to compare.

`run` computes them in plain torch operations (`own = False`) or through `accelerate_hpc_test_amd.ops` (`own = True`);
`exact` gives the same outputs in 64 bits. Sizes are those of the models that the framework ships or benchmarks
(hidden sizes 4096 to 7168, vocabularies 50257 to 128256, 8 experts) and generic ones around them.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
NORM_EPS = 1e-5
ROPE_TABLE = 32768  # positions in the cos / sin tables
IGNORE = -100


def listed():
    return [
        # layer norm -------------------------------------------------------------------------------------------------
        # one decoding step of 16 sequences through a block with hidden size 6144, residual add fused in
        {"name": "norm decode", "op": "norm", "rows": 16, "hidden": 6144, "dtype": "bf16", "residual": True, "train": False},
        # the norm of a training step at 8192 tokens, forward and backward, in the residual stream
        {"name": "norm train", "op": "norm", "rows": 8192, "hidden": 4096, "dtype": "bf16", "residual": True, "train": True},
        # an odd width and row count in 32 bits: an encoder's ragged batch, rows at no alignment
        {"name": "norm odd", "op": "norm", "rows": 3001, "hidden": 1027, "dtype": "fp32", "residual": False, "train": True},
        # rotary positions -------------------------------------------------------------------------------------------
        # one decoding step of 32 sequences at their own positions: 16 heads of 256, the first 64 rotated in pairs
        {"name": "rope decode", "op": "rope", "batch": 32, "seq": 1, "rot_heads": 32, "heads": 48, "dim": 256, "rotary": 64,
         "interleaved": True, "positions": True, "dtype": "bf16", "train": False},
        # a training sequence of 8192 tokens: 64 heads of 96, a quarter of each rotated in halves, forward and backward
        {"name": "rope train", "op": "rope", "batch": 1, "seq": 8192, "rot_heads": 128, "heads": 192, "dim": 96, "rotary": 24,
         "interleaved": False, "positions": False, "dtype": "bf16", "train": True},
        # prompts of an odd length in half precision, whole heads rotated in pairs
        {"name": "rope prompt", "op": "rope", "batch": 3, "seq": 1777, "rot_heads": 40, "heads": 48, "dim": 128, "rotary": 128,
         "interleaved": True, "positions": True, "dtype": "fp16", "train": False},
        # log-probabilities of given tokens ---------------------------------------------------------------------------
        # one decoding step of 16 sequences: the sampled tokens' log-probabilities and the 20 best alternatives
        {"name": "logprobs decode", "op": "logprobs", "rows": 16, "vocab": 128256, "top": 20, "dtype": "bf16",
         "temperature": 0.7, "train": False},
        # a policy step over 4096 tokens: log-probability and entropy, and the gradient of the logits
        {"name": "logprobs train", "op": "logprobs", "rows": 4096, "vocab": 128256, "top": 0, "dtype": "bf16",
         "temperature": 1.0, "train": True},
        # distillation on a ragged batch in 32 bits: an odd vocabulary, five alternatives that carry gradients
        {"name": "logprobs distil", "op": "logprobs", "rows": 777, "vocab": 50257, "top": 5, "dtype": "fp32",
         "temperature": 1.0, "train": True},
        # routing to experts -------------------------------------------------------------------------------------------
        # one decoding step of 64 sequences: 256 sigmoid-scored experts in 8 groups, a balance bias, 8 chosen
        {"name": "route decode", "op": "route", "rows": 64, "experts": 256, "top": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "fp32", "train": False},
        # the same router in training on 16384 tokens, forward and backward
        {"name": "route train", "op": "route", "rows": 16384, "experts": 256, "top": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "fp32", "train": True},
        # 8 softmax-scored experts, 2 chosen, on an odd number of tokens, with the router's logits in 16 bits
        {"name": "route softmax", "op": "route", "rows": 8191, "experts": 8, "top": 2, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renormalize": True, "scale": 1.0, "dtype": "bf16", "train": True},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "rope", "logprobs", "route"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if op == "norm":
        hidden = _log_uniform(rng, 48, 12288)
        if rng.random() < 0.6:
            hidden = (hidden + 7) // 8 * 8
        rows = _log_uniform(rng, 1, min(16384, 8192 * 4096 // hidden))
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "residual": rng.random() < 0.5, "train": train}
    if op == "rope":
        dim = rng.choice([48, 64, 80, 96, 128, 192, 256])
        rotary = rng.choice([dim, dim // 2, dim // 4 // 2 * 2, 2 * rng.randint(1, dim // 2)])
        kv = rng.choice([1, 2, 4, 8, 16])
        query = kv * rng.choice([1, 2, 4])
        heads = query + 2 * kv
        if rng.random() < 0.4:
            batch, seq = _log_uniform(rng, 1, 512), 1
        else:
            seq = _log_uniform(rng, 2, 8192)
            batch = rng.randint(1, max(1, min(8, 8192 * 192 * 96 // (seq * heads * dim))))
        return {"op": op, "batch": batch, "seq": seq, "rot_heads": query + kv, "heads": heads, "dim": dim, "rotary": rotary,
                "interleaved": rng.random() < 0.5, "positions": seq == 1 or rng.random() < 0.5, "dtype": dtype, "train": train}
    if op == "logprobs":
        vocab = _log_uniform(rng, 1000, 160000)
        rows = _log_uniform(rng, 1, min(4096, 2048 * 128256 // vocab))
        top = rng.choice([0, 0, 1, 5, 20, 32])
        if top:
            rows = min(rows, max(1, 512 * 128256 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.5]), "train": train}
    groups = rng.choice([1, 1, 4, 8])
    experts = groups * rng.randint(2, 48 if groups > 1 else 384)
    top_groups = rng.randint(1, groups)
    top = rng.randint(1, min(10, experts // groups * top_groups))
    return {"op": "route", "rows": _log_uniform(rng, 1, 16384), "experts": experts, "top": top,
            "scoring": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.5, "groups": groups,
            "top_groups": top_groups, "renormalize": top > 1 and rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]),
            "dtype": rng.choice(["fp32", "fp32", "bf16"]), "train": train}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _rope_tables(rotary, device):
    """cos / sin [positions, rotary / 2] of angles scaled linearly by 4 for long contexts, evaluated in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary) / 4.0
    angle = torch.outer(torch.arange(ROPE_TABLE, dtype=torch.float64, device=device), inv)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    dtype = DTYPES[case["dtype"]]
    op, st = case["op"], {"case": case}
    if op == "norm":
        rows, hidden = case["rows"], case["hidden"]
        # a residual stream: rows of different scale and a shared offset per channel
        spread = 1.0 + 0.2 * normal(hidden)
        x = (normal(rows, hidden) * spread + 0.3 * normal(hidden)) * (0.5 + normal(rows, 1).abs())
        st["x"] = x.to(dtype)
        st["residual"] = (2.0 * normal(rows, hidden)).to(dtype) if case["residual"] else None
        st["weight"] = (1.0 + 0.2 * normal(hidden)).to(dtype)
        st["bias"] = (0.2 * normal(hidden)).to(dtype)
        if case["train"]:
            st["dy"] = normal(rows, hidden).to(dtype)
            st["dres"] = normal(rows, hidden).to(dtype) if case["residual"] else None
        leaves = ("x", "residual", "weight", "bias")
    elif op == "rope":
        shape = (case["batch"], case["seq"], case["heads"], case["dim"])
        st["qkv"] = normal(*shape).to(dtype)
        st["cos"], st["sin"] = _rope_tables(case["rotary"], device)
        st["positions"] = None
        if case["positions"]:
            start = torch.randint(0, ROPE_TABLE - case["seq"] + 1, (case["batch"], 1), generator=g, device=device)
            st["positions"] = start + torch.arange(case["seq"], device=device)
        if case["train"]:
            st["dout"] = normal(*shape).to(dtype)
        leaves = ("qkv",)
    elif op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a trained model's logits: a broad body, and a few tokens per row far above it
        x = torch.empty(rows, vocab, device=device, dtype=dtype)
        for lo in range(0, rows, 512):
            part = normal(min(512, rows - lo), vocab).mul_(2.0)
            peaks = torch.randint(0, vocab, (part.shape[0], 24), generator=g, device=device)
            part.scatter_add_(1, peaks, 3.0 * normal(part.shape[0], 24) + 9.0)
            x[lo : lo + part.shape[0]] = part
            # a twelfth of the vocabulary is not allowed in every fifth row
            banned = torch.randint(0, vocab, (vocab // 12,), generator=g, device=device)
            x[lo : lo + part.shape[0] : 5, banned] = -math.inf
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=device)
        best = x.argmax(-1)
        likely = torch.rand(rows, generator=g, device=device) < 0.6
        allowed = x.gather(1, tokens[:, None])[:, 0] > -math.inf
        tokens = torch.where(likely | ~allowed, best, tokens)
        if case["train"]:  # prompts and padding carry no loss
            tokens = torch.where(torch.rand(rows, generator=g, device=device) < 0.1, torch.full_like(tokens, IGNORE), tokens)
            st["dlogprobs"] = normal(rows)
            st["dentropy"] = 0.1 * normal(rows)
            st["dtop"] = normal(rows, case["top"]) if case["top"] else None
        st["logits"], st["tokens"] = x, tokens
        leaves = ("logits",)
    else:
        rows, experts = case["rows"], case["experts"]
        st["logits"] = (normal(rows, experts) * 1.5 + 0.5 * normal(experts)).to(dtype)
        st["bias"] = 0.05 * normal(experts) if case["bias"] else None
        if case["train"]:
            st["dweights"] = normal(rows, case["top"])
        leaves = ("logits",)
    if case["train"]:
        for name in leaves:
            if st[name] is not None:
                st[name].requires_grad_()
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the operators in plain operations
# ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(st):
    case, dtype = st["case"], st["x"].dtype
    w, b = st["weight"].float(), st["bias"].float()
    x = st["x"].float()
    out = {}
    if case["residual"]:
        out["residual"] = (x + st["residual"].float()).to(dtype)
        x = out["residual"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + NORM_EPS)
    hat = centred * rstd
    out["y"] = (hat * w + b).to(dtype)
    if case["train"]:
        dy = st["dy"].float()
        dhat = dy * w
        dx = rstd * (dhat - dhat.mean(-1, keepdim=True) - hat * (dhat * hat).mean(-1, keepdim=True))
        if case["residual"]:
            dx = dx + st["dres"].float()
        out["dx"] = dx.to(dtype)
        if case["residual"]:
            out["dresidual"] = out["dx"]
        out["dweight"] = (dy * hat).sum(0).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


def _plain_rotate(x, cos, sin, case, positions):
    """x [B, S, heads, D] with its first `rotary` values rotated in heads [0, rot_heads); `sin` carries the direction."""
    rot, n = case["rotary"], case["rot_heads"]
    if positions is None:
        c, s = cos[: case["seq"], None], sin[: case["seq"], None]
    else:
        c, s = cos[positions][:, :, None], sin[positions][:, :, None]
    out = x.clone()
    part = x[:, :, :n, :rot].float()
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        out[:, :, :n, 0:rot:2] = (a * c - b * s).to(x.dtype)
        out[:, :, :n, 1:rot:2] = (b * c + a * s).to(x.dtype)
    else:
        a, b = part[..., : rot // 2], part[..., rot // 2 :]
        out[:, :, :n, : rot // 2] = (a * c - b * s).to(x.dtype)
        out[:, :, :n, rot // 2 : rot] = (b * c + a * s).to(x.dtype)
    return out


def _plain_rope(st):
    case = st["case"]
    out = {"out": _plain_rotate(st["qkv"], st["cos"], st["sin"], case, st["positions"])}
    if case["train"]:  # the gradient turns back by the same angles
        out["dqkv"] = _plain_rotate(st["dout"], st["cos"], -st["sin"], case, st["positions"])
    return out


def _best(x, k):
    """Indices of the k largest values of each row in falling order, equal values by rising index: 64-bit keys of the
    value's ordered bits above the complement of the index."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    at = torch.arange(x.shape[-1], device=x.device)
    return 0x7FFFFFFF - (torch.topk((bits << 32) | (0x7FFFFFFF - at), k, dim=-1)[0] & 0x7FFFFFFF)


def _plain_logprobs(st):
    case, logits, tokens = st["case"], st["logits"], st["tokens"]
    x = logits.float() * (1.0 / case["temperature"])
    counts = tokens != IGNORE
    at = tokens.clamp(min=0)[:, None]
    top = x.max(-1, keepdim=True)[0]
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    p = e / total
    finite = torch.where(x > -math.inf, x - top, torch.zeros_like(x))
    entropy = log_total - (p * finite).sum(-1, keepdim=True)
    zero = torch.zeros((), device=x.device)
    out = {"logprobs": torch.where(counts, (x.gather(1, at) - top - log_total)[:, 0], zero),
           "entropy": torch.where(counts, entropy[:, 0], zero)}
    if case["top"]:
        ids = _best(logits, case["top"])
        out["top_logprobs"] = torch.where(counts[:, None], x.gather(1, ids) - top - log_total, zero)
        out["top_tokens"] = torch.where(counts[:, None], ids, torch.full_like(ids, -1))
    if case["train"]:
        g, h = st["dlogprobs"][:, None], st["dentropy"][:, None]
        total_g = g + st["dtop"].sum(-1, keepdim=True) if case["top"] else g
        d = -p * (total_g + h * (finite - log_total + entropy))
        d.scatter_add_(1, at, g)
        if case["top"]:
            d.scatter_add_(1, ids, st["dtop"])
        d = d * (counts[:, None] / case["temperature"])
        out["dlogits"] = d.to(logits.dtype)
    return out


def _plain_route(st):
    case, logits = st["case"], st["logits"]
    experts, k, groups = case["experts"], case["top"], case["groups"]
    # scores in 64 bits: the choice turns on differences far under a 32-bit rounding of exp
    x = logits.double()
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + (-x).exp())
    else:
        e = (x - x.max(-1, keepdim=True)[0]).exp()
        score = e / e.sum(-1, keepdim=True)
    key = score if st["bias"] is None else score + st["bias"].double()
    if case["top_groups"] < groups:
        rating = torch.topk(key.view(-1, groups, experts // groups), 2, dim=-1)[0].sum(-1)
        chosen = torch.sort(rating, dim=-1, descending=True, stable=True)[1][:, : case["top_groups"]]
        open_ = torch.zeros_like(rating, dtype=torch.bool).scatter_(1, chosen, True)
        key = torch.where(open_.repeat_interleave(experts // groups, 1), key, torch.full_like(key, -math.inf))
    ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :k]
    score = score.float()
    s = score.gather(1, ids)
    total = s.sum(-1, keepdim=True) if case["renormalize"] else torch.ones_like(s[:, :1])
    share = s / total
    out = {"weights": share * case["scale"], "experts": ids}
    if case["train"]:
        u = st["dweights"] * case["scale"]
        ds = (u - (u * share).sum(-1, keepdim=True)) / total if case["renormalize"] else u
        if case["scoring"] == "sigmoid":
            d = torch.zeros_like(score).scatter_(1, ids, ds * s * (1.0 - s))
        else:
            d = torch.zeros_like(score).scatter_(1, ids, ds)
            d = score * (d - (ds * s).sum(-1, keepdim=True))
        out["dlogits"] = d.to(logits.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the same through the framework
# ---------------------------------------------------------------------------------------------------------------------
def _own_norm(st):
    from accelerate_hpc_test_amd.ops import layer_norm

    case = st["case"]
    y, res = layer_norm(st["x"], st["weight"], st["bias"], NORM_EPS, st["residual"])
    out = {"residual": res, "y": y} if case["residual"] else {"y": y}
    if case["train"]:
        if case["residual"]:
            grads = torch.autograd.grad((y, res), (st["x"], st["residual"], st["weight"], st["bias"]), (st["dy"], st["dres"]))
            out["dx"], out["dresidual"], out["dweight"], out["dbias"] = grads
        else:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    return out


def _own_rope(st):
    from accelerate_hpc_test_amd.ops import apply_rope

    case = st["case"]
    y = apply_rope(st["qkv"], st["cos"], st["sin"], case["rot_heads"], st["positions"], interleaved=case["interleaved"],
                   rotary_dim=case["rotary"])
    out = {"out": y}
    if case["train"]:
        (out["dqkv"],) = torch.autograd.grad(y, st["qkv"], st["dout"])
    return out


def _own_logprobs(st):
    from accelerate_hpc_test_amd.ops import token_logprobs

    case = st["case"]
    r = token_logprobs(st["logits"], st["tokens"], top_k=case["top"], temperature=case["temperature"], ignore_index=IGNORE)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    outputs, grads = [r.logprobs, r.entropy], [st.get("dlogprobs"), st.get("dentropy")]
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs, r.top_tokens
        outputs.append(r.top_logprobs)
        grads.append(st.get("dtop"))
    if case["train"]:
        (out["dlogits"],) = torch.autograd.grad(outputs, st["logits"], grads)
    return out


def _own_route(st):
    from accelerate_hpc_test_amd.ops import route_experts

    case = st["case"]
    w, ids = route_experts(st["logits"], case["top"], scoring=case["scoring"], bias=st["bias"], n_groups=case["groups"],
                           topk_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"])
    out = {"weights": w, "experts": ids}
    if case["train"]:
        (out["dlogits"],) = torch.autograd.grad(w, st["logits"], st["dweights"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rope": _own_rope, "logprobs": _own_logprobs, "route": _own_route}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "rope": _plain_rope, "logprobs": _plain_logprobs, "route": _plain_route}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size, train = BYTES[case["dtype"]], case["train"]
    if case["op"] == "norm":
        n, h = case["rows"] * case["hidden"], case["hidden"]
        tensors = (4 if case["residual"] else 2) + ((4 if case["residual"] else 2) if train else 0)
        return {"bytes": size * (tensors * n + (4 if train else 2) * h), "flops": (22 if train else 9) * n}
    if case["op"] == "rope":
        tokens = case["batch"] * case["seq"]
        n = tokens * case["heads"] * case["dim"]
        table = 4 * tokens * case["rotary"] + (8 * tokens if case["positions"] else 0)
        return {"bytes": (4 if train else 2) * size * n + table,
                "flops": (6 if train else 3) * tokens * case["rot_heads"] * case["rotary"]}
    if case["op"] == "logprobs":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        per_row = 16 + 12 * case["top"] + ((8 + 4 * case["top"]) if train else 0)
        return {"bytes": (2 if train else 1) * size * n + per_row * rows, "flops": (12 if train else 6) * n}
    n, rows = case["rows"] * case["experts"], case["rows"]
    per_row = 12 * case["top"] + (4 * case["top"] if train else 0)
    return {"bytes": (2 if train else 1) * size * n + per_row * rows + (4 * case["experts"] if case["bias"] else 0),
            "flops": (16 if train else 10) * n}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions: forward in torch's own functions, gradients by automatic differentiation
# ---------------------------------------------------------------------------------------------------------------------
def _exact_norm(st):
    case, dtype = st["case"], st["x"].dtype
    out = {}
    x = st["x"].detach().double()
    if case["residual"]:  # the stream is what is stored: the sum rounded to its type
        x = (x + st["residual"].detach().double()).to(dtype).double()
        out["residual"] = x
    leaf = x.clone().requires_grad_()
    w, b = (st[n].detach().double().requires_grad_() for n in ("weight", "bias"))
    var, mean = torch.var_mean(leaf, dim=-1, unbiased=False, keepdim=True)
    y = (leaf - mean) / torch.sqrt(var + NORM_EPS) * w + b
    out["y"] = y.detach()
    if case["train"]:
        dx, dw, db = torch.autograd.grad(y, (leaf, w, b), st["dy"].double())
        if case["residual"]:
            dx = dx + st["dres"].double()
            out["dresidual"] = dx
        out |= {"dx": dx, "dweight": dw, "dbias": db}
    return out


def _exact_rope(st):
    case, rot, n = st["case"], st["case"]["rotary"], st["case"]["rot_heads"]
    pos = st["positions"]
    if pos is None:
        pos = torch.arange(case["seq"], device=st["qkv"].device).expand(case["batch"], -1)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos].unsqueeze(2)

    def rotate(x, turn):
        x = x.detach().double()
        part = x[:, :, :n, :rot]
        shape = part.shape[:3]
        pair = part.reshape(*shape, rot // 2, 2) if case["interleaved"] else part.reshape(*shape, 2, rot // 2).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.reshape(*shape, rot) if case["interleaved"] else z.transpose(-1, -2).reshape(*shape, rot)
        return torch.cat([torch.cat([z, x[:, :, :n, rot:]], -1), x[:, :, n:]], 2)

    out = {"out": rotate(st["qkv"], turn)}
    if case["train"]:
        out["dqkv"] = rotate(st["dout"], turn.conj())
    return out


def _exact_logprobs(st):
    case = st["case"]
    parts = []
    for lo in range(0, case["rows"], 256):
        rows = slice(lo, min(lo + 256, case["rows"]))
        tokens = st["tokens"][rows]
        counts = tokens != IGNORE
        x = st["logits"].detach()[rows].double()
        z = (x / case["temperature"]).clone().requires_grad_()
        logp = torch.log_softmax(z, -1)
        # a banned token's term p log p is its limit, zero
        terms = torch.where(x > -math.inf, logp.exp() * logp.masked_fill(x == -math.inf, 0.0), torch.zeros_like(logp))
        part = {"logprobs": logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0] * counts, "entropy": -terms.sum(-1) * counts}
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, : case["top"]]
            part["top_logprobs"] = logp.gather(1, order) * counts[:, None]
            part["top_tokens"] = torch.where(counts[:, None], order, torch.full_like(order, -1))
        if case["train"]:
            loss = (part["logprobs"] * st["dlogprobs"][rows].double()).sum()
            loss = loss + (part["entropy"] * st["dentropy"][rows].double()).sum()
            if case["top"]:
                loss = loss + (part["top_logprobs"] * st["dtop"][rows].double()).sum()
            part["dlogits"] = torch.autograd.grad(loss, z)[0] / case["temperature"]
        parts.append({n: v.detach() for n, v in part.items()})
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_route(st):
    case = st["case"]
    x = st["logits"].detach().double().requires_grad_()
    score = torch.sigmoid(x) if case["scoring"] == "sigmoid" else torch.softmax(x, -1)
    key = score.detach() + (0.0 if st["bias"] is None else st["bias"].double())
    if case["top_groups"] < case["groups"]:
        size = case["experts"] // case["groups"]
        rating = torch.topk(key.unflatten(1, (case["groups"], size)), min(2, size), dim=-1)[0].sum(-1)
        closed = torch.sort(rating, dim=-1, descending=True, stable=True)[1][:, case["top_groups"] :]
        key.unflatten(1, (case["groups"], size)).scatter_(1, closed[..., None].expand(-1, -1, size), -math.inf)
    ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, : case["top"]]
    w = score.gather(1, ids)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * case["scale"]
    out = {"weights": w.detach(), "experts": ids}
    if case["train"]:
        (out["dlogits"],) = torch.autograd.grad(w, x, st["dweights"].double())
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "logprobs": _exact_logprobs, "route": _exact_route}[case["op"]](st)
