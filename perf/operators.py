"""Cases of the dropless mixture-of-experts operators and of the 8-bit AdamW step, in plain form and through the framework.

Operators, and what a pass returns:

* ``products``: ragged matrix products grouped by expert. Rows sorted by expert meet their expert's matrix:
  ``y[i] = x[i] W[e(i)]``; with ``grad`` also ``dx[i] = dy[i] W[e(i)]^T`` and ``dW[e] = sum_i x[i]^T dy[i]``. Rows after
  the last expert's belong to nobody: zero outputs, no gradient.
* ``mlp``: the SwiGLU experts over the same rows, ``(silu(x Wg) * (x Wu)) Wd``; with ``grad`` its four gradients.
* ``routing``: (token, choice) assignments sorted by expert (offsets, order and its inverse), the rows gathered into that
  order, the experts' rows summed back with the router's weights, and all gradients. An expert id outside the range is
  a dropped assignment: sorted last, a row of zeros, nothing in the sum.
* ``adamw``: an AdamW step over many tensors whose moments are held in 8 bits (e4m3) with a power-of-two scale for each
  256 elements of a tensor: the first moment, and the square root of the second. Rounding to 8 bits is stochastic, with
  a hash of (element, step) as the random number, so that moments which change little in a step still move on average.

Where ``own`` is false, ``run`` computes in 32 bits with elementary torch operations, rounding once to the outputs' type.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BLOCK = 256  # elements of a tensor that share the scale of a moment
_BETA1, _BETA2, _EPS, _LR, _DECAY = 0.9, 0.999, 1e-8, 1e-3, 1e-2
_MASK32 = 0xFFFFFFFF


def listed():
    return [
        # A step over a handful of tokens (8 tokens, two experts each): every expert's weights are read for a row or two.
        dict(name="products few rows bf16", op="products", rows=16, idle=0, experts=8, dim=768, out=1536, type="bf16", skew=0.5, grad=False),
        # The up projection of the repository's MoE benchmark (8 experts of 1536 over d_model 768, 64 x 1024 tokens, top 2), trained in bf16.
        dict(name="products moe bf16", op="products", rows=131072, idle=0, experts=8, dim=768, out=1536, type="bf16", skew=0.3, grad=True),
        # The same layer in the framework's default precision, a quarter of the tokens.
        dict(name="products moe fp32", op="products", rows=32768, idle=0, experts=8, dim=768, out=1536, type="fp32", skew=0.3, grad=True),
        # Many small experts with uneven loads.
        dict(name="products 64 experts bf16", op="products", rows=65536, idle=0, experts=64, dim=2048, out=1408, type="bf16", skew=0.8, grad=True),
        # Sizes that fit no tile, rows that nobody owns (dropped tokens), an expert that is rarely chosen.
        dict(name="products odd bf16", op="products", rows=4999, idle=130, experts=5, dim=515, out=771, type="bf16", skew=2.0, grad=True),
        # Experts of the repository's largest MLP (d_model 2048, hidden 5632).
        dict(name="mlp wide bf16", op="mlp", rows=32768, idle=0, experts=8, dim=2048, out=5632, type="bf16", skew=0.3, grad=True),
        # The MoE benchmark's experts in the default precision, a batch of 8 sequences.
        dict(name="mlp moe fp32", op="mlp", rows=16384, idle=0, experts=8, dim=768, out=1536, type="fp32", skew=0.3, grad=True),
        # Routing of a short batch: latency counts.
        dict(name="routing short bf16", op="routing", tokens=256, choices=2, experts=8, dim=768, type="bf16", drop=0.0, skew=0.3),
        # Routing of the MoE benchmark's whole batch.
        dict(name="routing moe bf16", op="routing", tokens=65536, choices=2, experts=8, dim=768, type="bf16", drop=0.0, skew=0.3),
        # fp32, an odd width, a tenth of the assignments dropped by a capacity limit.
        dict(name="routing odd fp32", op="routing", tokens=9001, choices=3, experts=17, dim=770, type="fp32", drop=0.1, skew=1.0),
        # The default tiny model of the examples: many tensors, hardly any elements.
        dict(name="adamw tiny model", op="adamw", layers=2, dim=64, hidden=65, experts=4, vocab=259, type="fp32"),
        # The MoE benchmark's model, 407 million parameters in 121 tensors.
        dict(name="adamw moe model", op="adamw", layers=12, dim=768, hidden=1536, experts=8, vocab=50304, type="fp32"),
    ]


def _between(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["products", "products", "mlp", "routing", "adamw"])
    kind = rng.choice(["bf16", "fp32"])
    if op in ("products", "mlp"):
        rows = _between(rng, 1, 32768)
        return dict(op=op, rows=rows, idle=rng.choice([0, _between(rng, 1, 200)]), experts=_between(rng, 1, 64), dim=_between(rng, 33, 2048),
                    out=_between(rng, 33, 2816), type=kind, skew=rng.uniform(0.0, 1.5), grad=rng.random() < 0.7)
    if op == "routing":
        experts = _between(rng, 2, 128)
        return dict(op=op, tokens=_between(rng, 1, 65536), choices=rng.randint(1, min(8, experts)), experts=experts, dim=_between(rng, 33, 2048),
                    type=kind, drop=rng.choice([0.0, rng.uniform(0.0, 0.5)]), skew=rng.uniform(0.0, 1.5))
    return dict(op=op, layers=rng.randint(1, 12), dim=_between(rng, 33, 768), hidden=_between(rng, 33, 1536), experts=rng.randint(1, 8),
                vocab=_between(rng, 100, 50304), type=kind)


# ------------------------------------------------------------------ inputs
def _sizes(case, seed):
    """Rows of each expert: a multinomial draw whose probabilities spread with ``skew``."""
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(case["skew"] * torch.randn(case["experts"], generator=g), 0)
    owners = torch.multinomial(p, case["rows"], replacement=True, generator=g)
    return torch.bincount(owners, minlength=case["experts"]).tolist()


def _shapes(case):
    """The tensors of a mixture-of-experts model."""
    d, h, e = case["dim"], case["hidden"], case["experts"]
    block = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (d, e), (e, d, h), (e, d, h), (e, h, d)]
    return [(case["vocab"], d)] + (block * case["layers"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    kind = _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] in ("products", "mlp"):
        rows, e, d, n = case["rows"] + case["idle"], case["experts"], case["dim"], case["out"]
        s["sizes"] = _sizes(case, seed)
        s["offsets"] = torch.tensor([0] + s["sizes"]).cumsum(0).to(device="cuda", dtype=torch.int32)
        s["x"] = normal(rows, d, dtype=kind)
        width = n if case["op"] == "products" else d
        s["dy"] = normal(rows, width, dtype=kind)
        names = {"w": (d, n)} if case["op"] == "products" else {"w_gate": (d, n), "w_up": (d, n), "w_down": (n, d)}
        s |= {name: normal(e, *shape, scale=math.sqrt(2 / sum(shape)), dtype=kind) for name, shape in names.items()}
        s["leaves"] = [s["x"]] + [s[name] for name in names]
        s["leaves"] = [t.requires_grad_(case["grad"]) for t in s["leaves"]]
    elif case["op"] == "routing":
        t, k, e, d = case["tokens"], case["choices"], case["experts"], case["dim"]
        scores = case["skew"] * normal(e) + normal(t, e)
        s["indices"] = torch.topk(scores, k, dim=1).indices
        dropped = torch.rand(t, k, device="cuda", generator=g) < case["drop"]
        s["indices"] = torch.where(dropped, torch.full_like(s["indices"], -1), s["indices"])
        w = torch.rand(t, k, device="cuda", generator=g) + 0.05
        s["weights"] = (w / w.sum(1, keepdim=True)).requires_grad_()
        s["x"] = normal(t, d, dtype=kind).requires_grad_()
        s["ys"] = normal(t * k, d, dtype=kind).requires_grad_()
        s["dxs"] = normal(t * k, d, dtype=kind)
        s["dout"] = normal(t, d, dtype=kind)
    else:
        numels = [math.prod(shape) for shape in _shapes(case)]
        blocks = [-(-n // _BLOCK) for n in numels]
        total = sum(blocks)
        # Blocks differ in size by powers of two; one in sixteen has seen no gradient yet (rows of an embedding).
        level = torch.exp2(torch.randint(-22, -13, (total,), device="cuda", generator=g).float())
        live = (torch.rand(total, device="cuda", generator=g) > 1 / 16).float()
        spread = (level * live)[:, None]
        # One flat buffer for each kind, every tensor at a whole number of blocks; element numbers restart with each tensor.
        s["element"] = torch.cat([torch.arange(b * _BLOCK, device="cuda", dtype=torch.int32) for b in blocks])
        inside = (s["element"] < torch.tensor(numels, device="cuda").repeat_interleave(torch.tensor(blocks, device="cuda") * _BLOCK)).view(total, _BLOCK)
        s["w"] = normal(total, _BLOCK, scale=0.02) * inside
        s["g"] = (normal(total, _BLOCK) * spread * 40 * inside).to(kind)
        s["m"] = (normal(total, _BLOCK).clamp(-6, 6) * 30 * live[:, None] * inside).to(torch.float8_e4m3fn)
        s["u"] = ((normal(total, _BLOCK).abs().clamp(max=6) * 30 + 1) * live[:, None] * inside).to(torch.float8_e4m3fn)
        s["m_scale"], s["u_scale"] = level.clone(), level.clone()
        s["step"] = 10
        del inside
        starts = torch.tensor([0] + blocks).cumsum(0).tolist()
        for key in ("w", "g", "m", "u"):
            s[key + "_list"] = [s[key].view(-1)[a * _BLOCK : a * _BLOCK + n].view(shape)
                                for a, n, shape in zip(starts, numels, _shapes(case))]
        for key in ("m_scale", "u_scale"):
            s[key + "_list"] = [s[key][a : a + b] for a, b in zip(starts, blocks)]
    return s


# ------------------------------------------------------------------ the operators
def run(s):
    return {"products": _products, "mlp": _mlp, "routing": _routing, "adamw": _adamw}[s["case"]["op"]](s)


def _per_expert(s, a, mats):
    """``a[rows of e] @ mats[e]`` for each expert, zeros in the rows that nobody owns."""
    parts = a.split(s["sizes"] + [s["case"]["idle"]])
    out = [p @ m for p, m in zip(parts, mats)]
    return torch.cat(out + [out[0].new_zeros(s["case"]["idle"], out[0].shape[1])])


def _per_expert_weights(s, a, b):
    """``a[rows of e]^T @ b[rows of e]`` for each expert."""
    return torch.stack([p.t() @ q for p, q in zip(a.split(s["sizes"] + [s["case"]["idle"]])[:-1], b.split(s["sizes"] + [s["case"]["idle"]])[:-1])])


def _products(s):
    if own:
        from abacus_b200.ops import experts

        y = experts.ragged_matmul(s["x"], s["w"], s["offsets"])
        return [y] + (list(torch.autograd.grad(y, s["leaves"], s["dy"])) if s["case"]["grad"] else [])
    with torch.no_grad():
        kind = s["x"].dtype
        x, w = s["x"].float(), s["w"].float()
        out = [_per_expert(s, x, w)]
        if s["case"]["grad"]:
            dy = s["dy"].float()
            out += [_per_expert(s, dy, w.transpose(1, 2)), _per_expert_weights(s, x, dy)]
        return [t.to(kind) for t in out]


def _mlp(s):
    if own:
        from abacus_b200.ops import experts

        y = experts.ragged_swiglu_mlp(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["offsets"])
        return [y] + (list(torch.autograd.grad(y, s["leaves"], s["dy"])) if s["case"]["grad"] else [])
    with torch.no_grad():
        kind = s["x"].dtype
        x, w_gate, w_up, w_down = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
        gate, up = _per_expert(s, x, w_gate), _per_expert(s, x, w_up)
        sig = 1 / (1 + torch.exp(-gate))
        h = gate * sig * up
        out = [_per_expert(s, h, w_down)]
        if s["case"]["grad"]:
            dy = s["dy"].float()
            dh = _per_expert(s, dy, w_down.transpose(1, 2))
            d_up = dh * gate * sig
            d_gate = dh * up * sig * (1 + gate * (1 - sig))
            dx = _per_expert(s, d_gate, w_gate.transpose(1, 2)) + _per_expert(s, d_up, w_up.transpose(1, 2))
            out += [dx, _per_expert_weights(s, x, d_gate), _per_expert_weights(s, x, d_up), _per_expert_weights(s, h, dy)]
        return [t.to(kind) for t in out]


def _routing(s):
    case = s["case"]
    if own:
        from abacus_b200.ops import experts

        plan = experts.expert_plan(s["indices"], case["experts"])
        xs = experts.dispatch_tokens(s["x"], plan)
        out = experts.combine_tokens(s["ys"], s["weights"], plan)
        grads = torch.autograd.grad((xs, out), (s["x"], s["ys"], s["weights"]), (s["dxs"], s["dout"]))
        return [plan.offsets, plan.order, plan.slot, xs, out, *grads]
    with torch.no_grad():
        t, k = s["indices"].shape
        kind = s["x"].dtype
        expert = s["indices"].reshape(-1)
        kept = (expert >= 0) & (expert < case["experts"])
        expert = torch.where(kept, expert, case["experts"])
        counts = (expert[:, None] == torch.arange(case["experts"], device=expert.device)).sum(0)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        order = torch.argsort(expert, stable=True)
        place = torch.empty_like(order)
        place[order] = torch.arange(t * k, device=order.device)
        live = kept[:, None].float()
        xs = s["x"].float()[order // k] * kept[order][:, None]
        ys = s["ys"].float()[place] * live  # the rows of each (token, choice), zero where dropped
        weights = s["weights"].reshape(-1, 1)
        dout = s["dout"].float().repeat_interleave(k, 0)
        out = (ys * weights).view(t, k, -1).sum(1)
        dx = (s["dxs"].float()[place] * live).view(t, k, -1).sum(1)
        dys = torch.empty_like(ys)
        dys[place] = dout * weights * live
        d_weights = (ys * dout).sum(1).view(t, k)
        slot = torch.where(kept, place, -1).view(t, k)
        return [offsets, order.to(torch.int32), slot.to(torch.int32), xs.to(kind), out.to(kind), dx.to(kind), dys.to(kind), d_weights]


def _noise(element, step):
    """32 random bits for each element and step: an integer hash, the same on every side."""
    x = (element.long() * 0x9E3779B1 + step * 0x7F4A7C15) & _MASK32
    x = ((x ^ (x >> 16)) * 0x6C62272F) & _MASK32
    x = ((x ^ (x >> 15)) * 0x2F0B4C47) & _MASK32
    return x ^ (x >> 16)


def _to_8_bits(value, noise16, positive):
    """(codes, scales) of one moment: e4m3 with a power-of-two scale a block, that puts the block's largest finite magnitude in
    [128, 256); rounded down, or up with the probability of the part that rounding down would lose."""
    finite = torch.isfinite(value)
    largest = torch.where(finite, value.abs(), 0.0).amax(1)
    exponent = ((largest.view(torch.int32) >> 23) - 7).clamp(min=1)
    scale = (exponent << 23).view(torch.float32)
    inverse = ((254 - exponent) << 23).view(torch.float32)
    a = value.abs() * inverse[:, None]
    base = torch.where(a < 2.0**-6, 2.0**-6, 0.0)  # below e4m3's smallest normal number its steps are all 2^-9
    bits = (a + base).view(torch.int32) + (noise16 << 4).to(torch.int32)
    q = (bits & -(1 << 20)).view(torch.float32) - base
    if positive:  # a second moment that is not zero stays so: the next step divides by its root
        q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
    q = torch.where(finite, torch.copysign(q, value), math.nan)
    return q.to(torch.float8_e4m3fn), scale


def _adamw(s):
    s["step"] += 1
    step = s["step"]
    keys = ("w", "m", "m_scale", "u", "u_scale")
    if own:
        from abacus_b200.ops import adamw8

        adamw8.step_(s["w_list"], s["g_list"], s["m_list"], s["m_scale_list"], s["u_list"], s["u_scale_list"],
                     lr=_LR, betas=(_BETA1, _BETA2), eps=_EPS, weight_decay=_DECAY, step=step)
        return {k: s[k] for k in keys}
    g = s["g"].float()
    m = s["m"].float() * s["m_scale"][:, None] * _BETA1 + g * (1 - _BETA1)
    u = s["u"].float() * s["u_scale"][:, None]
    u = torch.sqrt(u * u * _BETA2 + g * g * (1 - _BETA2))
    ratio = m / (u / math.sqrt(1 - _BETA2**step) + _EPS)
    s["w"].copy_(s["w"] * (1 - _LR * _DECAY) - ratio * (_LR / (1 - _BETA1**step)))
    noise = _noise(s["element"], step).view(m.shape)
    for key, value, bits in (("m", m, noise & 0xFFFF), ("u", u, noise >> 16)):
        q, scale = _to_8_bits(value, bits, key == "u")
        s[key].copy_(q)
        s[key + "_scale"].copy_(scale)
    return {k: s[k] for k in keys}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 2 if case.get("type") == "bf16" else 4
    if case["op"] in ("products", "mlp"):
        rows, idle, e, d, n = (case[k] for k in ("rows", "idle", "experts", "dim", "out"))
        mats = 1 if case["op"] == "products" else 3
        out = n if case["op"] == "products" else d
        used = min(e, rows)  # experts that own rows, at most
        flops = 2 * rows * d * n * mats
        nbytes = size * (rows * d + used * d * n * mats + (rows + idle) * out)
        if case["grad"]:
            flops *= 3
            nbytes += size * (rows * out + (rows + idle) * d + e * d * n * mats)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "routing":
        t, k, d = case["tokens"], case["choices"], case["dim"]
        kept = t * k * (1 - case["drop"])
        rows = size * d * (2 * t + 2 * t + 2 * kept + 2 * t * k)  # x, dx, out, dout; ys, dxs read; xs, dys written
        return {"bytes": rows + t * k * (8 + 4 + 4 + 4 + 4) + 4 * case["experts"], "flops": 6 * kept * d}
    n = sum(math.prod(shape) for shape in _shapes(case))
    return {"bytes": n * (8 + size + 4) + n // _BLOCK * 16, "flops": 20 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"products": _exact_products, "mlp": _exact_mlp, "routing": _exact_routing, "adamw": _exact_adamw}[case["op"]](s)


def _spans(s):
    ends = [int(v) for v in s["offsets"].tolist()]
    return list(enumerate(zip(ends[:-1], ends[1:])))


def _exact_products(s):
    x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
    y, dx, dw = x.new_zeros(x.shape[0], w.shape[2]), torch.zeros_like(x), torch.zeros_like(w)
    for e, (a, b) in _spans(s):
        y[a:b] = torch.einsum("sd,dn->sn", x[a:b], w[e])
        dx[a:b] = torch.einsum("sn,dn->sd", dy[a:b], w[e])
        dw[e] = torch.einsum("sd,sn->dn", x[a:b], dy[a:b])
    return [y, dx, dw] if s["case"]["grad"] else [y]


def _exact_mlp(s):
    """The gradients by torch's own differentiation of the formula, an expert at a time."""
    x = s["x"].detach().double()
    mats = [s[k].detach().double() for k in ("w_gate", "w_up", "w_down")]
    y, dx, dws = torch.zeros_like(x), torch.zeros_like(x), [torch.zeros_like(m) for m in mats]
    for e, (a, b) in _spans(s):
        with torch.enable_grad():
            parts = [x[a:b].clone().requires_grad_()] + [m[e].clone().requires_grad_() for m in mats]
            gate = parts[0] @ parts[1]
            ye = (gate * torch.sigmoid(gate) * (parts[0] @ parts[2])) @ parts[3]
        y[a:b] = ye.detach()
        if s["case"]["grad"]:
            grads = torch.autograd.grad(ye, parts, s["dy"][a:b].double())
            dx[a:b] = grads[0]
            for dw, got in zip(dws, grads[1:]):
                dw[e] = got
    return [y, dx, *dws] if s["case"]["grad"] else [y]


def _exact_routing(s):
    t, k = s["indices"].shape
    e = s["case"]["experts"]
    flat = s["indices"].reshape(-1).cpu()
    lists = [torch.nonzero(flat == i).reshape(-1) for i in range(e)] + [torch.nonzero((flat < 0) | (flat >= e)).reshape(-1)]
    order = torch.cat(lists)
    total = sum(len(v) for v in lists[:-1])
    offsets = [0]
    for v in lists[:-1]:
        offsets.append(offsets[-1] + len(v))
    slot = torch.full((t * k,), -1, dtype=torch.int64)
    slot[order[:total]] = torch.arange(total)
    x, ys, dxs, dout, w = (s[n].double() for n in ("x", "ys", "dxs", "dout", "weights"))
    used = order[:total].to(x.device)
    token = used // k
    xs, dys, dw = torch.zeros_like(ys), torch.zeros_like(ys), x.new_zeros(t * k)
    xs[:total] = x[token]
    flat_w = w.reshape(-1)[used]
    out = torch.zeros_like(x).index_add_(0, token, ys[:total] * flat_w[:, None])
    dx = torch.zeros_like(x).index_add_(0, token, dxs[:total])
    dys[:total] = dout[token] * flat_w[:, None]
    dw[used] = torch.einsum("sd,sd->s", ys[:total], dout[token])
    return [torch.tensor(offsets, dtype=torch.int32), order.to(torch.int32), slot.to(torch.int32).view(t, k), xs, out, dx, dys, dw.view(t, k)]


def _exact_adamw(s):
    step = s["step"] + 1
    g, w = s["g"].double(), s["w"].double()
    m = _BETA1 * (s["m"].double() * s["m_scale"].double()[:, None]) + (1 - _BETA1) * g
    v = _BETA2 * (s["u"].double() * s["u_scale"].double()[:, None]) ** 2 + (1 - _BETA2) * g * g
    u = v.sqrt()
    w = w - _LR * _DECAY * w - _LR * (m / (1 - _BETA1**step)) / ((v / (1 - _BETA2**step)).sqrt() + _EPS)
    out = {"w": w}
    noise = _noise(s["element"], step).view(m.shape)
    for key, value, bits in (("m", m, noise & 0xFFFF), ("u", u, noise >> 16)):
        # The scale that brings the block's largest magnitude to [128, 256), within 32 bits' normal numbers; then up or
        # down to a neighbour on the grid that 8 bits have there.
        largest = value.abs().amax(1)
        scale = torch.exp2((torch.floor(torch.log2(largest.clamp(min=1e-45))) - 7).clamp(min=-126.0))
        a = value.abs() / scale[:, None]
        grid = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
        q = torch.floor(a / grid + bits.double() / 65536) * grid
        if key == "u":
            q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
        out[key], out[key + "_scale"] = torch.sign(value) * q, scale
    return out
