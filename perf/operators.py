"""The operators of an MoE layer's training step, each as a case with its sizes:

  sort          tokens sorted by expert (every expert's rows padded to `align`), with the plan that leads back
  unsort        the sorted rows back in token order, summed with the routing weights
  sort_grad     the gradients of both: of the unsorted rows and the weights, and of the tokens
  act           SiLU(gate) * up with an 8-bit checkpoint of gate and up, and the backward pass from that checkpoint
  act_grad      the backward pass alone, from a checkpoint in hand
  rows          rows put into an 8-bit checkpoint and taken out again
  input_grad    gradient of the rows of a grouped product with packed weights
  weight_grad   gradient of the packed weights of a grouped product

With `own` false everything is computed with elementary torch operations in 32 bits, with `own`
true by the package's entry points.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128       # columns that share one scale of a checkpoint


def _package():
    path = os.path.join(os.getcwd(), "deepgemm-das_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import deepgemm
    return deepgemm


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step: top-8 of 256 experts, no padding (the compact layout)
        dict(name="sort one token", op="sort", tokens=1, top_k=8, experts=256, hidden=7168, align=1, dtype="bf16", dropped=0.0),
        # prefill of 4096 tokens over 32 local experts, every expert's block padded to 128 rows
        dict(name="sort prefill", op="sort", tokens=4096, top_k=8, experts=32, hidden=7168, align=128, dtype="bf16", dropped=0.0),
        # a decode batch whose experts live partly elsewhere (pairs without a row)
        dict(name="unsort decode batch", op="unsort", tokens=67, top_k=8, experts=256, hidden=7168, align=1, dtype="fp16", dropped=0.25),
        # a training micro-batch, backward through the way back and the way there
        dict(name="sort gradients", op="sort_grad", tokens=4095, top_k=8, experts=32, hidden=7168, align=128, dtype="bf16", dropped=0.0),
        # the experts' activation in a training step: forward, checkpoint, backward
        dict(name="activation e4m3", op="act", tokens=4096, top_k=8, experts=32, hidden=2048, align=128, dtype="bf16", kind="fp8", dropped=0.0),
        # the same with few, odd rows and an inner size that ends inside a scale block
        dict(name="activation small", op="act", tokens=37, top_k=1, experts=1, hidden=1000, align=1, dtype="fp16", kind="int8", dropped=0.0),
        # backward alone, as it runs long after the forward pass
        dict(name="activation backward", op="act_grad", tokens=4096, top_k=8, experts=32, hidden=2048, align=128, dtype="bf16", kind="fp8", dropped=0.0),
        # the rows that enter the experts, kept for the weight gradient in a byte each
        dict(name="rows int8", op="rows", tokens=16383, hidden=7168, dtype="bf16", kind="int8"),
        # gate and up projection of 32 experts, gradient of the sorted rows
        dict(name="input gradient", op="input_grad", tokens=4096, top_k=8, experts=32, n=4096, k=7168, align=128, dropped=0.0),
        # a short, ragged batch of small experts
        dict(name="input gradient small", op="input_grad", tokens=101, top_k=2, experts=8, n=336, k=704, align=128, dropped=0.0),
        # gate and up projection of 32 experts, gradient of the weights
        dict(name="weight gradient", op="weight_grad", tokens=4096, top_k=8, experts=32, n=4096, k=7168, align=128, dropped=0.0, dtype="bf16", accumulate=False),
        # small experts, added to a 32-bit gradient over micro-batches
        dict(name="weight gradient small", op="weight_grad", tokens=333, top_k=2, experts=4, n=336, k=576, align=128, dropped=0.0, dtype="fp32", accumulate=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "unsort", "sort_grad", "act", "act_grad", "rows", "input_grad", "weight_grad"])
    experts = _log(rng, 1, 256)
    top_k = rng.randint(1, min(8, experts))
    dropped = rng.choice([0.0, 0.0, 0.3])
    if op in ("sort", "unsort", "sort_grad"):
        hidden = _log(rng, 64, 7168)
        hidden = hidden if rng.random() < 0.25 else (hidden + 7) // 8 * 8
        return dict(op=op, tokens=_log(rng, 1, 16384 // top_k), top_k=top_k, experts=experts, hidden=hidden,
                    align=rng.choice([1, 16, 128, 256]) if experts <= 64 else 1, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), dropped=dropped)
    if op in ("act", "act_grad"):
        hidden = _log(rng, 64, 4096)
        hidden = hidden if rng.random() < 0.25 else (hidden + 7) // 8 * 8
        return dict(op=op, tokens=_log(rng, 1, 16384 // top_k), top_k=top_k, experts=experts, hidden=hidden, align=128 if experts <= 64 else 1,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), kind=rng.choice(["fp8", "int8"]), dropped=dropped)
    if op == "rows":
        hidden = _log(rng, 64, 7168)
        hidden = hidden if rng.random() < 0.25 else (hidden + 7) // 8 * 8
        return dict(op=op, tokens=_log(rng, 1, 16384), hidden=hidden, dtype=rng.choice(["bf16", "bf16", "fp16"]), kind=rng.choice(["fp8", "int8"]))
    experts = min(experts, 64)
    case = dict(op=op, tokens=_log(rng, 1, 8192 // min(top_k, experts)), top_k=min(top_k, experts), experts=experts,
                n=16 * _log(rng, 2, 256 if experts <= 32 else 64), k=64 * _log(rng, 1, 112 if experts <= 32 else 32), align=rng.choice([128, 256]), dropped=dropped)
    if op == "weight_grad":
        case["dtype"] = rng.choice(["bf16", "fp32"])
        case["accumulate"] = case["dtype"] == "fp32" and rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------ plans
def _capacity(case):
    """Rows that hold every expert's rows, padded."""
    pairs = case["tokens"] * case["top_k"]
    return (pairs + min(case["experts"], pairs) * (case["align"] - 1)) // case["align"] * case["align"]


def _sorting(ids, experts, align, cap):
    """(dest, m_indices, counts, offsets, m_total): where each pair (token, slot) goes when the pairs
    are sorted by expert, in their order, each expert's rows beginning at a multiple of `align`."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(experts + 1, dtype=torch.long, device=ids.device).index_add_(0, key, torch.ones_like(key))
    ends = counts.cumsum(0)
    blocks = (counts[:experts] + align - 1) // align * align
    offsets = blocks.cumsum(0) - blocks
    place = torch.arange(flat.numel(), device=ids.device) - (ends - counts)[key[order]]
    begin = torch.cat([offsets, offsets.new_zeros(1)])
    dest = torch.empty_like(key)
    dest[order] = begin[key[order]] + place
    dest = torch.where(key < experts, dest, -1)
    m_indices = torch.full((cap + 1,), -1, dtype=torch.int32, device=ids.device)
    m_indices[torch.where(dest < 0, cap, dest)] = torch.where(key < experts, key, -1).int()
    return (dest.view(ids.shape).int(), m_indices[:cap], counts[:experts].int(), offsets.int(), blocks.sum().view(1).int())


def _slots(m_indices, experts):
    """[experts, most rows of one] row numbers, `len(m_indices)` where an expert has fewer."""
    rows = m_indices.numel()
    key = torch.where(m_indices >= 0, m_indices.long(), experts)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=key.device).index_add_(0, key, torch.ones_like(key))
    order = torch.sort(key, stable=True).indices
    place = torch.arange(rows, device=key.device) - (counts.cumsum(0) - counts)[key[order]]
    most = max(1, int(counts[:experts].max()))
    slots = torch.full((experts + 1, max(most, int(counts.max()) + 1)), rows, dtype=torch.long, device=key.device)
    slots[key[order], place] = order
    return slots[:experts, :most].contiguous()


def _routing(case, gen):
    """Ids as a router gives them: distinct experts for a token, some experts liked more than others."""
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    liking = torch.randn(e, generator=gen, device=DEVICE) * 0.5
    scores = torch.rand(t, e, generator=gen, device=DEVICE).clamp_min(1e-9).log().neg().log().neg() + liking
    ids = torch.topk(scores, k, dim=1).indices
    gone = torch.rand(t, k, generator=gen, device=DEVICE) < case["dropped"]
    return torch.where(gone, -1, ids).to(torch.int32)


def _rows(gen, *shape, dtype=torch.bfloat16):
    """Activations: each row at a size of its own."""
    x = torch.randn(*shape, generator=gen, device=DEVICE)
    return (x * (0.5 + torch.rand(shape[0], 1, generator=gen, device=DEVICE))).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case=case)
    op = case["op"]
    dtype = TYPES[case.get("dtype", "bf16")]
    if op == "rows":
        s["x"] = _rows(gen, case["tokens"], case["hidden"], dtype=dtype)
        return s
    cap = _capacity(case)
    ids = _routing(case, gen)
    plan = _sorting(ids, case["experts"], case["align"], cap)
    m_indices = plan[1]
    if op == "sort":
        s["x"], s["ids"], s["cap"] = _rows(gen, case["tokens"], case["hidden"], dtype=dtype), ids, cap
        return s
    if op in ("unsort", "sort_grad"):
        s["plan"] = plan
        s["y"] = _rows(gen, cap, case["hidden"], dtype=dtype)
        weights = torch.rand(case["tokens"], case["top_k"], generator=gen, device=DEVICE) + 0.05
        s["weights"] = weights / weights.sum(1, keepdim=True)
        if op == "sort_grad":
            s["dout"] = _rows(gen, case["tokens"], case["hidden"], dtype=dtype)
            s["drows"] = _rows(gen, cap, case["hidden"], dtype=dtype)
        return s
    s["m_indices"] = m_indices
    if op in ("act", "act_grad"):
        x = _rows(gen, cap, 2 * case["hidden"], dtype=dtype)
        s["dact"] = _rows(gen, cap, case["hidden"], dtype=dtype)
        if op == "act":
            s["x"] = x
        else:
            s["q"], s["scale"] = _checkpoint(x.view(cap, 2, case["hidden"]), case["kind"])
            s["q"], s["scale"] = s["q"].view(cap, 2 * case["hidden"]), s["scale"].reshape(cap, -1)
        return s
    s["dy"] = _rows(gen, cap, case["n"])
    s["slots"] = _slots(m_indices, case["experts"])
    if op == "input_grad":
        s["w"] = (torch.randn(case["experts"], case["k"] // 64, case["n"], 64, generator=gen, device=DEVICE) / math.sqrt(case["k"])).bfloat16()
        return s
    s["x"] = _rows(gen, cap, case["k"])
    if case["accumulate"]:
        s["sum"] = torch.randn(case["experts"], case["k"] // 64, case["n"], 64, generator=gen, device=DEVICE)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _blocks(v):
    """[..., h] -> [..., blocks of BLOCK columns, BLOCK], the last one filled up with zeros."""
    h = v.shape[-1]
    return torch.nn.functional.pad(v, (0, -h % BLOCK)).unflatten(-1, (-1, BLOCK))


def _scale_of(amax, kind):
    """fp8: the smallest power of two that brings the block's largest value to 448 or less; int8: a
    127th of that value.  1 for a block of zeros, NaN for one that holds NaN or an infinity."""
    if kind == "fp8":
        m, e = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), (e - 8 - (m <= 0.875).int()).clamp_min(-126))
    else:
        scale = (amax / 127).clamp_min(2.0 ** -126)
    scale = torch.where(amax == 0, torch.ones_like(amax), scale)
    return torch.where(torch.isfinite(amax), scale, torch.full_like(amax, math.nan))


def _checkpoint(x, kind):
    """(q like x, scale [..., blocks])"""
    h = x.shape[-1]
    b = _blocks(x.float())
    scale = _scale_of(b.abs().amax(-1), kind)
    v = b / scale.unsqueeze(-1)
    q = v.to(torch.float8_e4m3fn) if kind == "fp8" else v.round().clamp(-127, 127).to(torch.int8)
    return q.flatten(-2)[..., :h].contiguous(), scale


def _restored(q, scale):
    h = q.shape[-1]
    return (_blocks(q.float()) * scale.unsqueeze(-1)).flatten(-2)[..., :h]


def _plain_act_grad(q, scale, dact, m_indices, dtype):
    m, h = dact.shape
    gate, up = _restored(q.view(m, 2, h), scale.view(m, 2, -1)).unbind(1)
    sig = 1 / (1 + torch.exp(-gate))
    d = dact.float()
    keep = (m_indices >= 0).unsqueeze(1)
    dgate = d * up * sig * (1 + gate * (1 - sig))
    dup = d * (gate * sig)
    act = gate * sig * up
    return (torch.where(keep, torch.cat([dgate, dup], 1), 0).to(dtype), torch.where(keep, act, 0).to(dtype))


def _plain(s):
    case = s["case"]
    op = case["op"]
    dtype = TYPES[case.get("dtype", "bf16")]
    if op == "sort":
        plan = _sorting(s["ids"], case["experts"], case["align"], s["cap"])
        rows = torch.zeros(s["cap"] + 1, case["hidden"], dtype=dtype, device=DEVICE)
        token = torch.arange(case["tokens"], device=DEVICE).repeat_interleave(case["top_k"])
        dest = plan[0].reshape(-1).long()
        rows[torch.where(dest < 0, s["cap"], dest)] = s["x"][token]
        return (rows[:s["cap"]],) + plan
    if op in ("unsort", "sort_grad"):
        dest = s["plan"][0].long()
        here = dest >= 0
        picked = s["y"][dest.clamp_min(0)].float()
        if op == "unsort":
            return torch.where(here.unsqueeze(2), picked * s["weights"].unsqueeze(2), 0).sum(1).to(dtype)
        dout = s["dout"].float().unsqueeze(1)
        cap = s["y"].shape[0]
        dy = torch.zeros(cap + 1, case["hidden"], dtype=dtype, device=DEVICE)
        dy[torch.where(here, dest, cap)] = (dout * s["weights"].unsqueeze(2)).to(dtype)
        dweights = torch.where(here, (dout * picked).sum(2), 0)
        dx = torch.where(here.unsqueeze(2), s["drows"][dest.clamp_min(0)].float(), 0).sum(1).to(dtype)
        return dy[:cap], dweights, dx
    if op == "rows":
        q, scale = _checkpoint(s["x"], case["kind"])
        return _restored(q, scale).to(dtype)
    if op == "act":
        x = s["x"]
        m, h = x.shape[0], case["hidden"]
        gate, up = x[:, :h].float(), x[:, h:].float()
        act = torch.where((s["m_indices"] >= 0).unsqueeze(1), gate / (1 + torch.exp(-gate)) * up, 0).to(dtype)
        q, scale = _checkpoint(x.view(m, 2, h), case["kind"])
        return (act,) + _plain_act_grad(q, scale, s["dact"], s["m_indices"], dtype)
    if op == "act_grad":
        return _plain_act_grad(s["q"], s["scale"], s["dact"], s["m_indices"], dtype)
    dy = torch.cat([s["dy"], s["dy"].new_zeros(1, case["n"])]).float()[s["slots"]]
    if op == "input_grad":
        w = s["w"].float().transpose(1, 2).flatten(2)
        dx = torch.zeros(s["dy"].shape[0] + 1, case["k"], dtype=torch.bfloat16, device=DEVICE)
        dx[s["slots"]] = torch.bmm(dy, w).bfloat16()
        return torch.where((s["m_indices"] >= 0).unsqueeze(1), dx[:-1], 0)
    x = torch.cat([s["x"], s["x"].new_zeros(1, case["k"])]).float()[s["slots"]]
    dw = torch.bmm(dy.transpose(1, 2), x).unflatten(2, (-1, 64)).transpose(1, 2)
    return (dw + s["sum"] if case["accumulate"] else dw).to(dtype).contiguous()


# ------------------------------------------------------------------------------------ the package's calls
def _own(s):
    dg = _package()
    case = s["case"]
    op = case["op"]
    if op == "sort":
        rows, plan = dg.sort_tokens(s["x"], s["ids"], case["experts"], align=case["align"])
        return (rows,) + tuple(plan)
    if op == "unsort":
        return dg.unsort_tokens(s["y"], dg.TokenPlan(*s["plan"]), s["weights"])
    if op == "sort_grad":
        plan = dg.TokenPlan(*s["plan"])
        dy, dweights = dg.unsort_tokens_grad(s["dout"], s["y"], plan, s["weights"])
        return dy, dweights, dg.sort_tokens_grad(s["drows"], plan)
    if op == "rows":
        return dg.restore_rows(dg.checkpoint_rows(s["x"], kind=case["kind"]))
    if op == "act":
        act, kept = dg.silu_mul_checkpoint(s["x"], kind=case["kind"], m_indices=s["m_indices"])
        return (act,) + tuple(dg.silu_mul_checkpoint_grad(kept, s["dact"], m_indices=s["m_indices"]))
    if op == "act_grad":
        kept = dg.Checkpoint(s["q"], s["scale"], TYPES[case["dtype"]])
        return tuple(dg.silu_mul_checkpoint_grad(kept, s["dact"], m_indices=s["m_indices"]))
    if op == "input_grad":
        return dg.grouped_bf16_input_grad(s["dy"], s["w"], s["m_indices"])
    if case["accumulate"]:
        # a step adds to the sum of the steps before; a copy keeps every pass the same
        return dg.grouped_bf16_weight_grad(s["dy"], s["x"], s["m_indices"], case["experts"], out=s["sum"].clone(), accumulate=True)
    return dg.grouped_bf16_weight_grad(s["dy"], s["x"], s["m_indices"], case["experts"], dtype=TYPES[case["dtype"]])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ what a pass needs
def work(case):
    """Each input read once and each output written once.  Of the sorted layouts, rows that stand
    for a pair are counted as inputs, and all of an output (its padding is zeros that are written)."""
    op = case["op"]
    size = SIZE[case.get("dtype", "bf16")]
    if op == "rows":
        values = case["tokens"] * case["hidden"]
        return {"bytes": 2 * values * size, "flops": 4 * values}
    pairs = case["tokens"] * case["top_k"]
    rows = max(1, round(pairs * (1 - case["dropped"])))
    cap = _capacity(case)
    if op == "sort":
        return {"bytes": (case["tokens"] + cap) * case["hidden"] * size + 8 * pairs + 4 * cap + 8 * case["experts"], "flops": pairs}
    if op == "unsort":
        return {"bytes": (case["tokens"] + rows) * case["hidden"] * size + 8 * pairs, "flops": 2 * rows * case["hidden"]}
    if op == "sort_grad":
        return {"bytes": (2 * case["tokens"] + 2 * rows + cap) * case["hidden"] * size + 12 * pairs, "flops": 4 * rows * case["hidden"]}
    if op == "act":      # in: gate, up, dact; out: act, dgate, dup, act again
        return {"bytes": (3 * rows + 4 * cap) * case["hidden"] * size, "flops": 30 * rows * case["hidden"]}
    if op == "act_grad":
        return {"bytes": (2 * rows + (rows + 3 * cap) * size) * case["hidden"] + 8 * rows * -(-case["hidden"] // BLOCK), "flops": 20 * rows * case["hidden"]}
    weights = case["experts"] * case["n"] * case["k"]
    flops = 2 * rows * case["n"] * case["k"]
    if op == "input_grad":
        used = min(case["experts"], max(1, rows))
        return {"bytes": 2 * (rows * case["n"] + cap * case["k"] + used * case["n"] * case["k"]), "flops": flops}
    out = weights * size * (2 if case["accumulate"] else 1)
    return {"bytes": 2 * rows * (case["n"] + case["k"]) + out, "flops": flops}


# ------------------------------------------------------------------------------------ in 64 bits
def _exact_kept(x, kind):
    """What an 8-bit checkpoint holds of the columns of x, as float64: block by block."""
    out = torch.empty_like(x, dtype=torch.float64)
    for c in range(0, x.shape[-1], BLOCK):
        v = x[..., c:c + BLOCK].double()
        top = v.abs().amax(-1, keepdim=True)
        if kind == "fp8":
            step = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp_min(1e-300) / 448) - 1e-13)), 1.0)
            out[..., c:c + BLOCK] = (v / step).to(torch.float8_e4m3fn).double() * step
        else:
            step = torch.where(top > 0, (top / 127).float().double(), 1.0)  # the scale is held in 32 bits
            out[..., c:c + BLOCK] = (v / step).float().round().clamp(-127, 127).double() * step
    return out


def _exact_act_grad(gate, up, dact, m_indices):
    s = torch.sigmoid(gate)
    d = dact.double()
    keep = (m_indices >= 0).double().unsqueeze(1)
    return (torch.cat([d * up * (s + gate * s * (1 - s)), d * gate * s], 1) * keep, gate * s * up * keep)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    dtype = TYPES[case.get("dtype", "bf16")]
    if op == "sort":
        rows = torch.zeros(s["cap"], case["hidden"], dtype=torch.float64, device=DEVICE)
        begin = 0
        for e in range(case["experts"]):
            token = (s["ids"] == e).nonzero()[:, 0]
            rows[begin:begin + len(token)] = s["x"][token].double()
            begin += -(-len(token) // case["align"]) * case["align"]
        return rows, None, None, None, None, None
    if op in ("unsort", "sort_grad"):
        dest = s["plan"][0]
        total = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=DEVICE)
        dx = torch.zeros_like(total)
        dy = torch.zeros(s["y"].shape, dtype=torch.float64, device=DEVICE)
        dweights = torch.zeros(dest.shape, dtype=torch.float64, device=DEVICE)
        for j in range(case["top_k"]):
            t = (dest[:, j] >= 0).nonzero()[:, 0]
            r = dest[t, j].long()
            w = s["weights"][t, j].double().unsqueeze(1)
            y = s["y"][r].double()
            total[t] += w * y
            if op == "sort_grad":
                d = s["dout"][t].double()
                dy[r] = w * d
                dweights[t, j] = torch.einsum("th,th->t", d, y)
                dx[t] += s["drows"][r].double()
        return total if op == "unsort" else (dy, dweights, dx)
    if op == "rows":
        return _exact_kept(s["x"], case["kind"])
    if op in ("act", "act_grad"):
        h = case["hidden"]
        if op == "act_grad":
            n = s["scale"].shape[1] // 2
            wide = s["scale"].double().view(-1, 2, n, 1).expand(-1, 2, n, BLOCK).reshape(-1, 2, n * BLOCK)[:, :, :h].reshape(-1, 2 * h)
            kept = s["q"].double() * wide
        else:
            kept = torch.cat([_exact_kept(s["x"][:, :h], case["kind"]), _exact_kept(s["x"][:, h:], case["kind"])], 1)
        back = _exact_act_grad(kept[:, :h], kept[:, h:], s["dact"], s["m_indices"])
        if op == "act_grad":
            return back
        gate, up = s["x"].double().chunk(2, 1)
        keep = (s["m_indices"] >= 0).double().unsqueeze(1)
        return (gate * torch.sigmoid(gate) * up * keep,) + back
    dy = s["dy"].double()
    if op == "input_grad":
        dx = torch.zeros(dy.shape[0], case["k"], dtype=torch.float64, device=DEVICE)
        for e in range(case["experts"]):
            r = (s["m_indices"] == e).nonzero()[:, 0]
            dx[r] = dy[r] @ s["w"][e].double().permute(1, 0, 2).reshape(case["n"], case["k"])
        return dx
    dw = torch.zeros(case["experts"], case["k"] // 64, case["n"], 64, dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        r = (s["m_indices"] == e).nonzero()[:, 0]
        dw[e] = (dy[r].T @ s["x"][r].double()).view(case["n"], -1, 64).permute(1, 0, 2)
    return dw + s["sum"].double() if case["accumulate"] else dw
