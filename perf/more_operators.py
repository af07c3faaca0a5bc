"""Products grouped by expert and products with 4-bit weights in groups: what they are timed on, and their plain forms.

A mixture-of-experts layer sends each of its tokens to `top` of `experts` experts. The picks - token t's j-th is number t * top + j - are put in the
order of their experts (stable), so that an expert's rows lie side by side, and every product runs over those groups of rows, whose lengths only the
GPU knows. A pick of no expert (id -1: padding) belongs to no group; what it would have written stays as it was.

A case is a plain dict. `op` says what a pass does:

  group    the picks in their experts' order: where each group begins, the picks, their tokens, and each pick's place (-1 where it has none)
  product  `flow` "up":   Y[i] = x[token of i] W_e^T   the tokens gathered on the way, W_e inter x hidden
                  "down": Y[i] = h[i] W_e^T            W_e hidden x inter
                  "back": dX[i] = dY[i] W_e            the gradient of "up" for its input
  weights  dW_e = sum over e's rows i of dY[i]^T x[token of i], the gradient of "up" for its weights; zero for an expert that nobody picked
  u4       Y[i] = x[token of i] W_e^T, W_e[j][p] = (code - zero) * scale: codes of four bits, a scale and a zero point for every `group_k` values of a row;
           one expert and top 1: an ordinary layer
"""
import math

import torch

own = False


def _case(name, op, **sizes):
    return {"name": name, "op": op, **sizes}


def listed():
    return [
        # The choice of a decode batch: latency.
        _case("group 16 tokens 8 of 128", "group", tokens=16, top=8, experts=128, idle=0),
        # The choice of a long prefill or a training batch with padding at its end.
        _case("group 16384 tokens 8 of 256", "group", tokens=16384, top=8, experts=256, idle=100),
        # A decode batch through the first projection of small experts: their weights are what is read.
        _case("up 32 tokens 4 of 32", "product", flow="up", tokens=32, top=4, experts=32, hidden=2048, inter=2816, dtype="bf16", out="same", idle=0),
        # Prefill through a few large experts; the largest.
        _case("up 4096 tokens 2 of 8", "product", flow="up", tokens=4096, top=2, experts=8, hidden=4096, inter=14336, dtype="bf16", out="same", idle=0),
        # Prefill through the second projection of many small experts.
        _case("down 4096 tokens 8 of 64", "product", flow="down", tokens=4096, top=8, experts=64, hidden=2048, inter=1408, dtype="bf16", out="f32", idle=0),
        # Training: the input's gradient there.
        _case("back 4096 tokens 8 of 64", "product", flow="back", tokens=4096, top=8, experts=64, hidden=2048, inter=1408, dtype="f16", out="same", idle=0),
        # No size a multiple of anything, padding at the batch's end.
        _case("up 1001 tokens 3 of 20 odd", "product", flow="up", tokens=1001, top=3, experts=20, hidden=2077, inter=1443, dtype="bf16", out="f32", idle=13),
        # Training: the weights' gradient of a few large experts.
        _case("weights 4096 tokens 2 of 8", "weights", tokens=4096, top=2, experts=8, hidden=4096, inter=4096, dtype="bf16", out="f32", idle=0),
        # ... and of many small ones, some of which hardly anybody picks.
        _case("weights 1024 tokens 6 of 64", "weights", tokens=1024, top=6, experts=64, hidden=2048, inter=1408, dtype="f16", out="same", idle=0),
        # One token through an ordinary layer with 4-bit weights.
        _case("u4 1x4096x11008", "u4", tokens=1, top=1, experts=1, hidden=4096, inter=11008, group_k=128, zeros=True, dtype="bf16", out="f32", idle=0),
        # A decode batch through a large layer, short groups without zero points.
        _case("u4 16x8192x8192", "u4", tokens=16, top=1, experts=1, hidden=8192, inter=8192, group_k=32, zeros=False, dtype="f16", out="same", idle=0),
        # A decode batch through experts with 4-bit weights.
        _case("u4 8 tokens 4 of 32", "u4", tokens=8, top=4, experts=32, hidden=2048, inter=2816, group_k=64, zeros=True, dtype="bf16", out="same", idle=0),
    ]


def _log_uniform(rng, low, high):
    return min(max(round(math.exp(rng.uniform(math.log(low), math.log(high)))), low), high)


def _size(rng, low, high, step=64):
    """Log-uniform; four of five multiples of `step`, the others as they fall."""
    v = _log_uniform(rng, low, high)
    return max(step, v // step * step) if rng.random() < 0.8 else v


def draw(rng):
    op = rng.choice(("group", "product", "product", "product", "weights", "u4", "u4"))
    experts = _log_uniform(rng, 2, 256)
    top = rng.randint(1, min(8, experts))
    if op == "group":
        tokens = _log_uniform(rng, 1, 65536)
        return {"op": op, "tokens": tokens, "top": top, "experts": experts, "idle": rng.choice((0, 0, tokens // 8))}
    dtype, out = rng.choice(("bf16", "bf16", "f16")), rng.choice(("f32", "same"))
    if op == "u4":
        if rng.random() < 0.5:
            experts, top = 1, 1
        while True:
            hidden, inter = 32 * _log_uniform(rng, 8, 448), _size(rng, 256, 14336)
            if experts * hidden * inter <= 8 * 4096 * 14336:
                return {"op": op, "tokens": _log_uniform(rng, 1, 64), "top": top, "experts": experts, "hidden": hidden, "inter": inter,
                        "group_k": rng.choice((32, 64, 128, 128)), "zeros": rng.random() < 0.5, "dtype": dtype, "out": out, "idle": 0}
    while True:
        tokens, hidden, inter = _log_uniform(rng, 1 if op == "product" else 64, 16384), _size(rng, 256, 7168), _size(rng, 256, 14336)
        if experts * hidden * inter <= 8 * 4096 * 14336 and tokens * top * hidden * inter <= 8192 * 4096 * 14336 and tokens * top * max(hidden, inter) <= 1 << 28:
            break
    case = {"op": op, "tokens": tokens, "top": top, "experts": experts, "hidden": hidden, "inter": inter, "dtype": dtype, "out": out, "idle": rng.choice((0, 0, tokens // 8))}
    if op == "product":
        case["flow"] = rng.choice(("up", "down", "back"))
    return case


# ---------------------------------------------------------------------------------------------------------------------
# the operators in their plain form
# ---------------------------------------------------------------------------------------------------------------------

def _plain_group(ids, top, experts):
    picks = ids.flatten().long()
    keys, order = torch.sort(torch.where(picks >= 0, picks, torch.full_like(picks, experts)), stable=True)  # those of no expert come last
    offsets = torch.searchsorted(keys, torch.arange(experts + 1, device=ids.device))
    position = torch.arange(len(picks), device=ids.device)
    inside = position < offsets[-1]
    place = torch.empty_like(order)
    place[order] = torch.where(inside, position, torch.full_like(position, -1))
    return tuple(v.int() for v in (offsets, torch.where(inside, order, torch.full_like(order, -1)), torch.where(inside, order // top, torch.full_like(order, -1)), place))


def _plain_weights(s, e):
    """Expert e's weights in 32 bits."""
    if s["op"] != "u4":
        return s["w"][e].float()
    codes = s["codes"][e]
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float()
    part = s["group_k"]
    scale = s["scales"][e].float().repeat_interleave(part, dim=-1)[:, :q.shape[1]]
    zero = s["zero"][e].float().repeat_interleave(part, dim=-1)[:, :q.shape[1]] if s["zero"] is not None else 8.0
    return (q - zero) * scale


def _plain(s):
    op = s["op"]
    if op == "group":
        return _plain_group(s["ids"], s["top"], s["experts"])
    rows, dtype = s["rows"].long(), s["x"].dtype
    kept = torch.float32 if s["out"] == "f32" else dtype
    parts, first = [], 0
    if op == "weights":
        for size in s["sizes"]:
            part = rows[first:first + size]
            parts.append((s["dy"][first:first + size].float().t() @ s["x"][part].float()).to(kept))
            first += size
        return torch.stack(parts)
    a = s["x"][rows.clamp(min=0)] if s["gather"] else s["x"]
    for e, size in enumerate(s["sizes"]):
        if size:
            w = _plain_weights(s, e)
            parts.append((a[first:first + size].float() @ (w if op == "product" and s["flow"] == "back" else w.t())).to(kept))
        first += size
    parts.append(torch.zeros((s["picks"] - first, s["n"]), dtype=kept, device=a.device))
    return torch.cat(parts)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _normal(gen, shape, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen)


def _choice(gen, case):
    """The experts of every token: the largest of logits in which some experts are more popular than others."""
    t, e = case["tokens"], case["experts"]
    ids = torch.topk(_normal(gen, (t, e)) + _normal(gen, (1, e), 0.7), case["top"], dim=-1).indices.int()
    if case["idle"]:
        ids[t - case["idle"]:] = -1
    return ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, s = case["op"], dict(case)
    ids = _choice(gen, case)
    if op == "group":
        s["ids"] = ids
        return s
    # The grouping, which a program has from the layer's router.
    offsets, _, rows, _ = _plain_group(ids, case["top"], case["experts"])
    s["offsets"], s["rows"], s["picks"] = offsets, rows, case["tokens"] * case["top"]
    s["sizes"] = (offsets[1:] - offsets[:-1]).tolist()
    h, i, e, dtype = case["hidden"], case["inter"], case["experts"], _TYPES[case["dtype"]]
    flow = case.get("flow", "up")
    s["gather"] = flow == "up"
    s["k"], s["n"] = (h, i) if flow == "up" else (i, h)
    s["x"] = _normal(gen, (case["tokens"] if s["gather"] else s["picks"], s["k"])).to(dtype)
    if op == "weights":
        s["dy"] = _normal(gen, (s["picks"], i), 0.02).to(dtype)
        return s
    shape = (h, i) if flow == "down" else (i, h)
    if op == "product":
        s["w"] = torch.empty((e, *shape), dtype=dtype, device="cuda")
        for j in range(e):
            s["w"][j] = _normal(gen, shape, 1.0 / math.sqrt(s["k"]))
        return s
    part = case["group_k"]
    blocks = -(-h // part)
    s["codes"] = torch.empty((e, i, h // 2), dtype=torch.uint8, device="cuda")
    s["scales"] = torch.empty((e, i, blocks), dtype=dtype, device="cuda")
    s["zero"] = torch.empty((e, i, blocks), dtype=torch.uint8, device="cuda") if case["zeros"] else None
    for j in range(e):
        w = torch.nn.functional.pad(_normal(gen, (i, h), 1.0 / math.sqrt(h)), (0, blocks * part - h)).view(i, blocks, part)
        low, high = w.amin(dim=-1).clamp(max=0.0), w.amax(dim=-1).clamp(min=0.0)
        scale = ((high - low) / 15 if case["zeros"] else torch.maximum(high, -low) / 7).clamp(min=1e-4).to(dtype)
        zero = torch.round(-low / scale.float()).clamp(0, 15) if case["zeros"] else torch.full_like(low, 8.0)
        q = (torch.round(w / scale.float().unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).view(i, -1)[:, :h]
        s["codes"][j], s["scales"][j] = q[:, 0::2] | (q[:, 1::2] << 4), scale
        if case["zeros"]:
            s["zero"][j] = zero.to(torch.uint8)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the operators through the library
# ---------------------------------------------------------------------------------------------------------------------

_ready = None


def _library():
    """The library, bound to torch's stream; every buffer is device memory, so no pointer needs to be looked up."""
    global _ready
    if _ready is None:
        import skl_amd
        lib = skl_amd.load()
        if lib.skl_hip_init(torch.cuda.current_device()) != 0:
            skl_amd.check_error()
        lib.skl_hip_set_pointer_mode(1)
        lib.skl_hip_set_stream(torch.cuda.current_stream().cuda_stream)
        _ready = lib
    return _ready


def _plan(s):
    """The call of a pass and its outputs: buffers that the program keeps."""
    lib, op, e = _library(), s["op"], s["experts"]
    if op == "group":
        count = s["tokens"] * s["top"]
        out = (torch.empty(e + 1, dtype=torch.int32, device="cuda"), *(torch.full((count,), -1, dtype=torch.int32, device="cuda") for _ in range(3)))
        offsets, order, rows, place = (t.data_ptr() for t in out)
        return lib.skl_group_rows_gfx950, (count, s["ids"].data_ptr(), s["top"], e, offsets, order, rows, place), out, None
    kind, single = s["dtype"], s["out"] == "f32"
    result = "f32" if single else kind
    x, k, n, m = s["x"], s["k"], s["n"], s["picks"]
    rows = (s["rows"].data_ptr() if s["gather"] else None, x.shape[0])
    dtype = torch.float32 if single else x.dtype
    offsets = s["offsets"].data_ptr()
    if e == 1:  # an ordinary layer: all rows are one group, as they lie
        offsets, rows = None, (None, m)
    if op == "weights":
        out = torch.zeros((e, s["inter"], s["hidden"]), dtype=dtype, device="cuda")
        entry = getattr(lib, f"skl_gemm_groupedk_{kind}c_{kind}_{result}_gfx950")
        args = (e, offsets, s["inter"], s["hidden"], m, 1.0, s["dy"].data_ptr(), s["inter"], None, m, x.data_ptr(), s["hidden"], *rows,
                0.0, out.data_ptr(), s["hidden"], s["inter"] * s["hidden"])
        return entry, args, out, None
    out = torch.zeros((m, n), dtype=dtype, device="cuda")
    if op == "u4":
        from skl_amd import U4Weights
        blocks = s["scales"].shape[-1]
        w = U4Weights(group_k=s["group_k"], codes=s["codes"].data_ptr(), ld=k, expert=n * k, scales=s["scales"].data_ptr(),
                      zeros=s["zero"].data_ptr() if s["zero"] is not None else None, ld_scales=blocks, expert_scales=n * blocks)
        entry = getattr(lib, f"skl_gemm_grouped_{kind}_u4c_{result}_gfx950")
        return entry, (e, offsets, m, n, k, 1.0, x.data_ptr(), k, *rows, w, 0.0, out.data_ptr(), n), out, w
    entry = getattr(lib, f"skl_gemm_grouped_{kind}_{kind}rc_{result}_gfx950")
    strides = (n, 1) if s["flow"] == "back" else (1, k)
    return entry, (e, offsets, m, n, k, 1.0, x.data_ptr(), k, *rows, s["w"].data_ptr(), *strides, n * k, 0.0, out.data_ptr(), n), out, None


def run(state):
    if not own:
        return _plain(state)
    if "plan" not in state:
        state["plan"] = _plan(state)
    entry, args, out, _ = state["plan"]
    entry(*args)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# work, and the results in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    t, top, e = case["tokens"], case["top"], case["experts"]
    live, picks = t - case["idle"], t * top
    if case["op"] == "group":
        return {"bytes": 4 * (picks + 3 * picks + e + 1), "flops": 0}
    h, i, m = case["hidden"], case["inter"], live * top
    reached = e * (1 - (1 - top / e) ** live)  # experts that some token chooses, on average
    size, flow = 4 if case["out"] == "f32" else 2, case.get("flow", "up")
    tokens = 2 * live * h
    if case["op"] == "weights":
        return {"bytes": tokens + 2 * m * i + size * e * h * i, "flops": 2 * m * h * i}
    if case["op"] == "u4":
        part = case["group_k"]
        return {"bytes": tokens + reached * i * (h / 2 + -(-h // part) * (3 if case["zeros"] else 2)) + size * m * i, "flops": 2 * m * h * i}
    moved = {"up": tokens + size * m * i, "down": 2 * m * i + size * m * h, "back": 2 * m * i + size * m * h}[flow]
    return {"bytes": moved + 2 * reached * h * i, "flops": 2 * m * h * i}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "group":
        return None  # whole numbers
    starts = s["offsets"].tolist()
    x, rows = s["x"], s["rows"].long()
    if op == "weights":
        out = torch.zeros((s["experts"], s["inter"], s["hidden"]), dtype=torch.float64, device="cuda")
        for e, (b, f) in enumerate(zip(starts, starts[1:])):
            if f > b:
                torch.mm(s["dy"][b:f].double().t(), x.double().index_select(0, rows[b:f]), out=out[e])
        return out
    y = torch.zeros((s["picks"], s["n"]), dtype=torch.float64, device="cuda")
    for e, (b, f) in enumerate(zip(starts, starts[1:])):
        if f == b:
            continue
        a = x.index_select(0, rows[b:f]).double() if s["gather"] else x[b:f].double()
        if op == "u4":
            codes = s["codes"][e]
            w = torch.empty((s["n"], s["k"]), dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (codes % 16).double(), (codes // 16).double()
            group = torch.arange(s["k"], device="cuda") // s["group_k"]
            w -= s["zero"][e].double()[:, group] if s["zero"] is not None else 8
            w *= s["scales"][e].double()[:, group]
        else:
            w = s["w"][e].double()
        y[b:f] = a @ (w if op == "product" and s["flow"] == "back" else w.t())
    return y
