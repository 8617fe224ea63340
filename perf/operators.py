"""What the language-model operators of metalgym_b200 are measured on.

Six entry points in four groups: controls on logits (penalties for repeated
actions, biases, action masks) and their gradient, the draw from controlled
logits, the clipped PPO loss of controlled logits with its gradient, and the
orthogonalised (Newton-Schulz) update alone and inside a whole optimiser step.

`own` selects the framework's kernels; otherwise every operator is computed in
elementary torch operations in 32 bits (64 for the race of the draw, whose
winner is a whole number). `exact` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CODES = {"f32": 0, "bf16": 1, "f16": 2}
_NS = (3.4445, -4.7750, 2.0315)  # the quintic's coefficients
_M32 = 0xFFFFFFFF


# ------------------------------------------------------------------ cases


def _logits(op, name, rows, actions, dtype, pad=0, mask="row", bias="none", history=0, ret=False, scores="penalties"):
    return {"name": name, "op": op, "rows": rows, "actions": actions, "pad": pad, "dtype": dtype, "mask": mask,
            "bias": bias, "history": history, "ret": ret, "scores": scores}


def _matrices(op, name, batch, rows, cols, dtype="f32", nesterov=True, clip=True):
    return {"name": name, "op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype, "nesterov": nesterov,
            "clip": clip}


def listed():
    return [
        # one sequence's next-action scores in a constrained decode: latency
        _logits("control", "control one row 32768", 1, 32768, "bf16", bias="shared", history=512),
        # a full serving batch with every control in use
        _logits("control", "control 256 x 131072", 256, 131072, "bf16", bias="shared", history=2048),
        # the gradient of a training batch through the controls; an odd action set, so rows start off alignment
        _logits("control_backward", "control gradient 1000 x 50001", 1000, 50001, "f16", history=777),
        # 4096 environments with six actions in the framework's 64-column head, invalid actions masked
        _logits("sample", "draw 4096 x 6", 4096, 6, "bf16", pad=58, history=0, ret=True),
        # a serving batch drawn straight from the logits
        _logits("sample", "draw 512 x 131072", 512, 131072, "bf16", bias="shared", history=1024),
        # the framework's own minibatch: 4096 rows, six actions, value column, masks
        _logits("loss", "loss 4096 x 6", 4096, 6, "bf16", pad=58, ret=True),
        # a token-level minibatch
        _logits("loss", "loss 4096 x 32768", 4096, 32768, "bf16", mask="none"),
        # fp32 logits of an odd action set with every control
        _logits("loss", "loss 1000 x 50001", 1000, 50001, "f32", bias="shared", history=300),
        # the up projections of two blocks (embed 128, hidden 512)
        _matrices("muon", "muon step 2 x 128 x 512", 2, 128, 512),
        # the down projections of four blocks at embed 512, hidden 2048
        _matrices("muon", "muon step 4 x 2048 x 512", 4, 2048, 512),
        # an odd matrix alone, from 16-bit gradients
        _matrices("orthogonalize", "orthogonalize 333 x 1001", 1, 333, 1001, dtype="bf16"),
        # a large square matrix, where the tensor cores bound it
        _matrices("orthogonalize", "orthogonalize 4096 x 4096", 1, 4096, 4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("control", "control_backward", "sample", "loss", "muon", "orthogonalize"))
    if op in ("muon", "orthogonalize"):
        batch = rng.choice((1, 1, 2, 3, 4, 8))
        rows, cols = _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)
        while batch * min(rows, cols) ** 2 * max(rows, cols) > 4096 ** 3:
            batch = max(1, batch // 2)
        case = _matrices(op, "", batch, rows, cols, rng.choice(("f32", "bf16", "f16")) if op == "orthogonalize" else "f32",
                         rng.random() < 0.7, rng.random() < 0.7)
    else:
        cap = {"control": 256 * 131072, "control_backward": 1000 * 50001, "sample": 512 * 131072, "loss": 1000 * 50001}[op]
        actions = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(8192, cap // (2 * actions))))
        case = _logits(op, "", rows, actions, rng.choice(("f32", "bf16", "f16")), rng.choice((0, 0, 1, 3, 8, 58)),
                       rng.choice(("row", "row", "shared", "none")), rng.choice(("none", "shared", "row")),
                       rng.choice((0, _log_int(rng, 1, 2048))), op in ("sample", "loss") and rng.random() < 0.3,
                       rng.choice(("penalties", "repetition", "frequency")))
        if case["ret"] and not case["pad"]:
            case["pad"] = 1  # the value column stands behind the last action
    del case["name"]
    return case


def work(case):
    if "batch" in case:
        s, n = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        per = 22 if case["op"] == "muon" else 2 + _TYPES[case["dtype"]].itemsize
        return {"bytes": case["batch"] * s * n * per, "flops": case["batch"] * 5 * (3 * s * s * n + s ** 3)}
    r, a, size = case["rows"], case["actions"], _TYPES[case["dtype"]].itemsize
    passes = {"control": 2, "control_backward": 3 if case["history"] and case["scores"] != "frequency" else 2, "sample": 1, "loss": 2}[case["op"]]
    words = (a + 31) // 32
    small = 4 * words * {"row": r, "shared": 1, "none": 0}[case["mask"]] + 4 * r * case["history"]
    if case["op"] != "control_backward":
        small += 4 * a * {"row": r, "shared": 1, "none": 0}[case["bias"]]
    small += {"control": 0, "control_backward": 0, "sample": 20 * r, "loss": 36 * r}[case["op"]]
    return {"bytes": passes * r * a * size + small, "flops": 10 * r * a}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if "batch" in case:
        b, m, n = case["batch"], case["rows"], case["cols"]
        # a policy gradient: a few strong directions over a noise floor
        rank = max(1, min(m, n) // 8)

        def gradient():
            return 1e-3 * (torch.bmm(normal(b, m, rank), normal(b, rank, n)) / math.sqrt(rank) + 0.3 * normal(b, m, n))

        s = {"case": case, "grad": gradient().to(_TYPES[case["dtype"]])}
        if case["op"] == "muon":
            s["momentum"] = 5.0 * gradient()
            s["master"] = normal(b, m, n) / math.sqrt(m)
            s["weights"] = s["master"].bfloat16()
            # partial sums of the squared gradient norm, as the gradient sums leave them
            s["norms"] = s["grad"].square().flatten(1).sum(1)
            s["max_norm"] = 0.5 * float(s["norms"].sum().sqrt()) if case["clip"] else 0.0
            s["lr"], s["scale"], s["decay"], s["wd"] = 3e-4, 0.2 * math.sqrt(max(m, n)), 0.95, 0.01
        else:
            s["out"] = torch.empty(b, m, n, dtype=torch.bfloat16, device="cuda")
        return s

    r, a = case["rows"], case["actions"]
    ld, kind = a + case["pad"], _TYPES[case["dtype"]]
    s = {"case": case, "logits": (3.0 * normal(r, ld)).to(kind)}
    words = (a + 31) // 32
    mask_rows = {"row": r, "shared": 1, "none": 0}[case["mask"]]
    if mask_rows:
        # grammars leave anything from a few actions to nearly all of them
        share = torch.tensor([0.05, 0.5, 0.95], device="cuda")[torch.randint(0, 3, (mask_rows, 1), generator=g, device="cuda")]
        bits = uniform(mask_rows, words * 32) < share
        bits.scatter_(1, torch.randint(0, a, (mask_rows, 1), generator=g, device="cuda"), True)
        if mask_rows > 8:
            bits[mask_rows // 2] = False  # a dead end: nothing is allowed
        place = torch.arange(32, device="cuda")
        value = (bits.reshape(mask_rows, words, 32).long() << place).sum(2)
        s["mask"] = torch.where(value > 0x7FFFFFFF, value - (1 << 32), value).int()
    bias_rows = {"row": r, "shared": 1, "none": 0}[case["bias"]]
    if bias_rows:
        s["bias"] = normal(bias_rows, a)
    if case["history"]:
        h = case["history"]
        s["history"] = (uniform(r, h) ** 3 * a).int().clamp_(max=a - 1)  # some actions often, most never
        s["lengths"] = torch.randint(0, h + 1, (r,), generator=g, device="cuda").int()
        if case["scores"] in ("penalties", "repetition"):
            s["repetition"] = 1.0 + 0.3 * uniform(r)
        if case["scores"] in ("penalties", "frequency"):
            s["frequency"], s["presence"] = 0.4 * uniform(r), 0.6 * uniform(r)
    if case["op"] == "control":
        s["out"] = torch.empty(r, ld, dtype=kind, device="cuda")
    elif case["op"] == "control_backward":
        s["dy"] = (normal(r, ld) / 64).to(kind)
        s["out"] = torch.empty(r, ld, dtype=kind, device="cuda")
    elif case["op"] == "sample":
        s["rng"] = torch.randint(-(1 << 31), 1 << 31, (r,), generator=g, device="cuda").int()
        s["rng"][s["rng"] == 0] = 1
        s["action"] = torch.empty(r, dtype=torch.int32, device="cuda")
        s["log_prob"], s["entropy"], s["value"] = (torch.empty(r, device="cuda") for _ in range(3))
    else:
        act = (uniform(r) * a).int().clamp_(max=a - 1)
        if mask_rows:  # mostly actions that the mask allows, as a draw gives them
            allowed = torch.where(_allowed(s, a), uniform(mask_rows, a), torch.full((), -1.0, device="cuda")).argmax(1).int()
            act = allowed.expand(r).contiguous()
        act[uniform(r) < 0.02] = -1  # padding
        s["action"] = act
        # the old policy's log-probability of the action under the same controls
        x, _ = _control(s, a)
        near = x.gather(1, act.long().clamp(min=0)[:, None])[:, 0] - x.logsumexp(1)
        s["old"] = torch.where(near.isfinite(), near, torch.zeros((), device="cuda")) + 0.1 * normal(r)
        s["adv"], s["returns"] = normal(r), normal(r)
        s["adv_stats"] = torch.stack((s["adv"].mean(), 1 / (s["adv"].std(unbiased=False) + 1e-8)))
        s["grad"] = torch.empty(r, ld, dtype=kind, device="cuda")
        s["stats"] = torch.empty(r, 5, device="cuda")
    return s


def _allowed(s, actions):
    """The mask's bits as truth values [rows or 1][actions]."""
    at = torch.arange(actions, device="cuda")
    return (s["mask"][:, at // 32] >> (at % 32)) & 1 != 0


# ------------------------------------------------------------------ plain forms


def _counts(s, rows, actions):
    """How often each action stands in the row's history, [rows][actions] fp32."""
    h = s["history"].long()
    valid = (torch.arange(h.shape[1], device="cuda") < s["lengths"][:, None]) & (h >= 0) & (h < actions)
    return torch.zeros(rows, actions, device="cuda").scatter_add_(1, h.clamp(0, actions - 1), valid.float())


def _control(s, actions):
    """The controlled logits in fp32 and the factor of their gradient."""
    x = s["logits"][:, :actions].float()
    factor = None
    if "history" in s:
        n = _counts(s, x.shape[0], actions)
        seen = n > 0
        if "repetition" in s:
            rep = s["repetition"][:, None]
            factor = torch.where(seen, torch.where(x > 0, 1 / rep, rep), torch.ones((), device="cuda"))
            x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        if "frequency" in s:
            x = torch.where(seen, (x - s["frequency"][:, None] * n) - s["presence"][:, None], x)
    if "bias" in s:
        x = x + s["bias"]
    if "mask" in s:
        x = torch.where(_allowed(s, actions), x, torch.full((), -math.inf, device="cuda"))
    return x, factor


def _first_best(key):
    """The lowest index of each row's largest key; -1 where every key is -inf."""
    best = key.amax(1, keepdim=True)
    at = torch.arange(key.shape[1], device="cuda")
    first = torch.where(key == best, at, key.shape[1]).amin(1)
    return torch.where(best[:, 0] > -math.inf, first, -1)


def _next_word(word):
    w = word.long() & _M32
    w = w ^ ((w << 13) & _M32)
    w = w ^ (w >> 17)
    return w ^ ((w << 5) & _M32)


def _signed(w):
    return torch.where(w > 0x7FFFFFFF, w - (1 << 32), w).int()


def _race(words, actions):
    """Exponential(1) times of every action, 64 bits, from the rows' words."""
    h = (words[:, None] + torch.arange(actions, device="cuda") * 0x9E3779B9) & _M32
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & _M32
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & _M32
    h = h ^ (h >> 16)
    return -torch.log1p(-(h.double() + 0.5) * 2.0 ** -32)


def _run_control(s):
    a = s["case"]["actions"]
    if own:
        mg, c, stream = _own(s)
        x, out = s["logits"], s["out"]
        mg.call("mg_logits_control", x.data_ptr(), _CODES[s["case"]["dtype"]], x.shape[1], c, out.data_ptr(), out.shape[1],
                x.shape[0], a, stream)
        return out[:, :a]
    return _control(s, a)[0].to(s["logits"].dtype)


def _run_control_backward(s):
    a = s["case"]["actions"]
    if own:
        mg, c, stream = _own(s)
        x, dy, out = s["logits"], s["dy"], s["out"]
        mg.call("mg_logits_control_backward", x.data_ptr(), _CODES[s["case"]["dtype"]], x.shape[1], c, dy.data_ptr(),
                dy.shape[1], out.data_ptr(), out.shape[1], x.shape[0], a, stream)
        return out[:, :a]
    dx = s["dy"][:, :a].float()
    x = s["logits"][:, :a].float()
    if "history" in s and "repetition" in s:
        rep = s["repetition"][:, None]
        dx = torch.where(_counts(s, x.shape[0], a) > 0, torch.where(x > 0, dx / rep, dx * rep), dx)
    if "mask" in s:
        dx = torch.where(_allowed(s, a), dx, torch.zeros((), device="cuda"))
    return dx.to(s["logits"].dtype)


def _run_sample(s):
    a, with_value = s["case"]["actions"], s["case"]["ret"]
    if own:
        mg, c, stream = _own(s)
        x = s["logits"]
        mg.call("mg_logits_sample", x.data_ptr(), _CODES[s["case"]["dtype"]], x.shape[1], c, s["rng"].data_ptr(),
                s["action"].data_ptr(), s["log_prob"].data_ptr(), s["entropy"].data_ptr(),
                s["value"].data_ptr() if with_value else None, x.shape[0], a, stream)
        out = {"action": s["action"], "log_prob": s["log_prob"], "entropy": s["entropy"], "rng": s["rng"]}
        return dict(out, value=s["value"]) if with_value else out
    x, _ = _control(s, a)
    words = _next_word(s["rng"])
    s["rng"].copy_(_signed(words))
    action = _first_best(x.double() - torch.log(_race(words, a)))
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1)
    chosen = x.gather(1, action.clamp(min=0)[:, None])[:, 0]
    some = action >= 0
    zero = torch.zeros((), device="cuda")
    log_prob = torch.where(some, (chosen - top[:, 0]) - torch.log(total), zero)
    below = torch.where(e > 0, e * (x - top), zero).sum(1)
    entropy = torch.where(some, torch.log(total) - below / total, zero)
    out = {"action": action.int(), "log_prob": log_prob, "entropy": entropy, "rng": s["rng"]}
    return dict(out, value=s["logits"][:, a].float()) if with_value else out


_CLIP, _VALUE, _ENTROPY = 0.2, 0.5, 0.01


def _run_loss(s):
    a, ret = s["case"]["actions"], s["case"]["ret"]
    rows = s["logits"].shape[0]
    if own:
        mg, c, stream = _own(s)
        x, d = s["logits"], s["grad"]
        mg.call("mg_logits_policy_loss", x.data_ptr(), _CODES[s["case"]["dtype"]], x.shape[1], c, s["action"].data_ptr(),
                s["adv"].data_ptr(), s["adv_stats"].data_ptr(), s["returns"].data_ptr() if ret else None,
                s["old"].data_ptr(), d.data_ptr(), d.shape[1], s["stats"].data_ptr(), rows, a, _CLIP, _VALUE, _ENTROPY,
                1.0 / rows, stream)
        return {"grad": d[:, : a + 1] if ret else d[:, :a], "stats": s["stats"]}
    x, factor = _control(s, a)
    action = s["action"].long()
    chosen = x.gather(1, action.clamp(min=0)[:, None])[:, 0]
    live = (action >= 0) & (chosen > -math.inf)
    zero = torch.zeros((), device="cuda")
    top = torch.where(live, x.amax(1), zero)[:, None]
    log_p = (x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True))
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, zero).sum(1)
    log_a = torch.where(live, log_p.gather(1, action.clamp(min=0)[:, None])[:, 0], zero)
    ratio = torch.exp(log_a - s["old"])
    adv = (s["adv"] - s["adv_stats"][0]) * s["adv_stats"][1]
    one, two = ratio * adv, ratio.clamp(1 - _CLIP, 1 + _CLIP) * adv
    slope = torch.where(one <= two, -adv * ratio, zero)
    hit = torch.arange(a, device="cuda") == action[:, None]
    dl = slope[:, None] * (hit.float() - p) + torch.where(p > 0, _ENTROPY * p * (log_p + entropy[:, None]), zero)
    dl = torch.where(live[:, None], dl * (1.0 / rows), zero)
    if factor is not None:
        dl = dl * factor
    columns = [-torch.minimum(one, two), zero.expand(rows), entropy, s["old"] - log_a, ((ratio - 1).abs() > _CLIP).float()]
    if ret:
        err = s["logits"][:, a].float() - s["returns"]
        columns[1] = 0.5 * _VALUE * err * err
        dl = torch.cat((dl, torch.where(live, _VALUE * err * (1.0 / rows), zero)[:, None]), 1)
    stats = torch.where(live[:, None], torch.stack(columns, 1), zero)
    return {"grad": dl.to(s["logits"].dtype), "stats": stats}


def _newton_schulz(u, steps=5):
    norm = u.flatten(1).norm(dim=1)[:, None, None]
    x = torch.where(norm > 0, u / norm, torch.zeros((), device="cuda"))
    flip = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if flip else x
    for _ in range(steps):
        gram = torch.bmm(x, x.transpose(1, 2))
        x = _NS[0] * x + torch.bmm(_NS[1] * gram + _NS[2] * torch.bmm(gram, gram), x)
    return x.transpose(1, 2) if flip else x


def _run_orthogonalize(s):
    u = s["grad"]
    if own:
        mg, _, stream = _own(s)
        b, m, n = u.shape
        out, space = s["out"], _workspace(s, mg)
        mg.call("mg_orthogonalize", u.data_ptr(), _CODES[s["case"]["dtype"]], n, m * n, out.data_ptr(), 1, n, m * n, b, m, n, 5,
                space.data_ptr(), space.numel(), stream)
        return out
    return _newton_schulz(u.float()).bfloat16()


def _run_muon(s):
    nesterov = s["case"]["nesterov"]
    if own:
        mg, _, stream = _own(s)
        b, m, n = s["grad"].shape
        space = _workspace(s, mg)
        mg.call("mg_muon_step", s["master"].data_ptr(), s["grad"].data_ptr(), s["momentum"].data_ptr(), s["weights"].data_ptr(),
                m * n, b, m, n, s["norms"].data_ptr(), s["norms"].numel(), s["max_norm"], s["lr"], s["scale"], s["decay"],
                int(nesterov), s["wd"], 5, None, space.data_ptr(), space.numel(), stream)
        return {"master": s["master"], "momentum": s["momentum"], "weights": s["weights"]}
    g = s["grad"]
    if s["max_norm"] > 0:
        norm = s["norms"].sum().sqrt()
        g = g * torch.where(norm > s["max_norm"], s["max_norm"] / (norm + 1e-6), torch.ones((), device="cuda"))
    s["momentum"].mul_(s["decay"]).add_(g)
    u = g + s["decay"] * s["momentum"] if nesterov else s["momentum"]
    s["master"].mul_(1 - s["lr"] * s["wd"]).sub_((s["lr"] * s["scale"]) * _newton_schulz(u))
    s["weights"].copy_(s["master"])
    return {"master": s["master"], "momentum": s["momentum"], "weights": s["weights"]}


def _own(s):
    """The framework, the state's control descriptor (device pointers that the program keeps) and the stream."""
    import ctypes

    import metalgym_b200 as mg

    if "logits" in s and "controls" not in s:
        def at(key):
            return s[key].data_ptr() if key in s else None

        s["descriptor"] = mg.LogitControls(
            mask=at("mask"), mask_stride=s["mask"].shape[1] if s["case"]["mask"] == "row" else 0,
            bias=at("bias"), bias_stride=s["bias"].shape[1] if s["case"]["bias"] == "row" else 0,
            history=at("history"), history_stride=s["case"]["history"], history_len=at("lengths"), history_max=s["case"]["history"],
            repetition=at("repetition"), frequency=at("frequency"), presence=at("presence"))
        s["controls"] = ctypes.addressof(s["descriptor"])
    return mg, s.get("controls"), torch.cuda.current_stream().cuda_stream


def _workspace(s, mg):
    """The optimiser's workspace, kept by the program."""
    if "workspace" not in s:
        import ctypes

        need = ctypes.c_size_t()
        b, m, n = s["grad"].shape
        mg.call("mg_muon_workspace", b, m, n, ctypes.byref(need))
        s["workspace"] = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    return s["workspace"]


_RUN = {"control": _run_control, "control_backward": _run_control_backward, "sample": _run_sample, "loss": _run_loss,
        "orthogonalize": _run_orthogonalize, "muon": _run_muon}


def run(state):
    return _RUN[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_control(s, a):
    """Controlled logits, whether each is allowed, and the derivative to the raw ones, row by row of the definition."""
    x = s["logits"][:, :a].double()
    rows = x.shape[0]
    slope = torch.ones_like(x)
    if "history" in s:
        width, h = s["history"].shape[1], s["history"].long()
        inside = torch.arange(width, device="cuda").expand(rows, width) < s["lengths"].long()[:, None]
        flat = (torch.arange(rows, device="cuda")[:, None] * a + h)[inside & (h >= 0) & (h < a)]
        n = torch.bincount(flat, minlength=rows * a).reshape(rows, a).double()
        if "repetition" in s:
            rep = s["repetition"].double()[:, None].expand_as(x)
            hit = n > 0
            slope[hit & (x > 0)] = (1 / rep)[hit & (x > 0)]
            slope[hit & (x <= 0)] = rep[hit & (x <= 0)]
            x = x * slope
        if "frequency" in s:
            x = x - s["frequency"].double()[:, None] * n - s["presence"].double()[:, None] * (n > 0)
    if "bias" in s:
        x = x + s["bias"].double()
    allowed = torch.ones_like(x, dtype=torch.bool)
    if "mask" in s:
        bits = (s["mask"].long()[:, :, None] >> torch.arange(32, device="cuda")).remainder(2)
        allowed = bits.flatten(1)[:, :a].bool().expand(rows, a)
        x = x.masked_fill(~allowed, -math.inf)
        slope = slope.masked_fill(~allowed, 0.0)
    return x, allowed, slope


def exact(case, seed):
    s = prepare(case, seed)
    if "batch" in case:
        g = s["grad"].double()
        if case["op"] == "muon":
            if case["clip"]:
                norm = float(s["norms"].double().sum().sqrt())
                if norm > s["max_norm"]:
                    g = g * (s["max_norm"] / (norm + 1e-6))
            momentum = s["decay"] * s["momentum"].double() + g
            u = momentum * s["decay"] + g if case["nesterov"] else momentum
        else:
            u = g
        done = []
        for one in u:
            x = one / one.norm()
            if x.shape[0] > x.shape[1]:
                for _ in range(5):
                    gram = x.t() @ x
                    x = x @ (_NS[0] * torch.eye(gram.shape[0], device="cuda", dtype=torch.float64) + _NS[1] * gram + _NS[2] * (gram @ gram))
            else:
                for _ in range(5):
                    gram = x @ x.t()
                    x = (_NS[0] * torch.eye(gram.shape[0], device="cuda", dtype=torch.float64) + _NS[1] * gram + _NS[2] * (gram @ gram)) @ x
            done.append(x)
        o = torch.stack(done)
        if case["op"] == "orthogonalize":
            return o
        master = s["master"].double() * (1 - s["lr"] * s["wd"]) - s["lr"] * s["scale"] * o
        return {"master": master, "momentum": momentum, "weights": master}
    a = case["actions"]
    x, allowed, slope = _exact_control(s, a)
    if case["op"] == "control":
        return x
    if case["op"] == "control_backward":
        return torch.where(allowed, s["dy"][:, :a].double() * slope, 0.0)
    rows = x.shape[0]
    if case["op"] == "sample":
        action = (x - _race(_next_word(s["rng"]), a).log()).argmax(1)
    else:
        action = s["action"].long()
    live = allowed.any(1) & (action >= 0) & allowed.gather(1, action.clamp(min=0)[:, None])[:, 0]
    x = torch.where(live[:, None], x, 0.0)
    log_p = torch.log_softmax(x, 1)
    p = log_p.exp()
    entropy = torch.special.entr(p).sum(1)
    log_a = log_p.gather(1, action.clamp(min=0)[:, None])[:, 0]
    if case["op"] == "sample":
        out = {"action": None, "log_prob": torch.where(live, log_a, 0.0), "entropy": torch.where(live, entropy, 0.0), "rng": None}
        return dict(out, value=s["logits"][:, a].double()) if case["ret"] else out
    old, stats = s["old"].double(), s["adv_stats"].double()
    adv = (s["adv"].double() - stats[0]) * stats[1]
    ratio = (log_a - old).exp()
    inside = torch.minimum(ratio * adv, ratio.clamp(1 - _CLIP, 1 + _CLIP) * adv)
    slope_a = torch.where(ratio * adv <= inside, -adv * ratio, 0.0)
    d = -slope_a[:, None] * p
    d.scatter_add_(1, action.clamp(min=0)[:, None], slope_a[:, None])
    d = d + _ENTROPY * (entropy[:, None] * p - torch.special.entr(p))
    d = torch.where(live[:, None], d * slope / rows, 0.0)
    value = torch.zeros_like(adv)
    if case["ret"]:
        err = s["logits"][:, a].double() - s["returns"].double()
        value = 0.5 * _VALUE * err ** 2
        d = torch.cat((d, torch.where(live, _VALUE * err / rows, 0.0)[:, None]), 1)
    rows5 = torch.stack((-inside, value, entropy, old - log_a, ((ratio - 1).abs() > _CLIP).double()), 1)
    return {"grad": d, "stats": torch.where(live[:, None], rows5, 0.0)}
