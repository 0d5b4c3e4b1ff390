"""Measured cases of the gated linear recurrence (whole sequences, training pass, single token) and of the AdamW step over
many tensors (states in 32 or 8 bits).

``run`` computes an operator in its plain form (elementary torch operations) or, where ``own`` is true, through this package's
entry points.  ``exact`` restates the definitions in 64 bits.

The recurrence: a = sigmoid(f); h_t = a_t h_{t-1} + (1 - a_t) z_t; y_t = sigmoid(o_t) h_t, or h_t without an output gate.
Positions at or behind a row's length give y = 0 and leave the state alone; ``reverse`` runs from the row's last position
to its first.

AdamW: g' = gs g with gs = grad_scale clip / max(|grad_scale g|, clip) over all tensors; m' = b1 m + (1 - b1) g';
v' = b2 v + (1 - b2) g'^2; p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps).  States in 8 bits: m and
sqrt(v) as e4m3 values times a power of two for each 128 elements, rounded stochastically by a word that is a function of
(seed, step, element); a root above zero is never rounded to zero.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 128                                                    # elements that share a scale; tensors start at multiples of it
ADAM = {"lr": 2e-4, "b1": 0.9, "b2": 0.999, "eps": 1e-8, "clip": 1.0, "seed": 1234, "step": 20}


# ---- cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one direction of a text encoder on a synthesis batch: short, ragged, fp32 -- launches and latency count
        {"name": "scan_text_f32", "kind": "scan", "dtype": "f32", "B": 32, "T": 140, "H": 256, "gate": False, "ragged": True, "reverse": True},
        # a batch of 800-frame utterances at the encoder's full width: the ordinary size
        {"name": "scan_frames_bf16", "kind": "scan", "dtype": "bf16", "B": 32, "T": 800, "H": 512, "gate": True, "ragged": True, "reverse": False},
        # two long recordings or documents: few rows, the time axis has to be split
        {"name": "scan_long_bf16", "kind": "scan", "dtype": "bf16", "B": 2, "T": 65536, "H": 1024, "gate": True, "ragged": False, "reverse": False},
        # training passes (forward, then backward) of the same three uses; the long one has an odd length and width
        {"name": "train_text_f32", "kind": "train", "dtype": "f32", "B": 32, "T": 140, "H": 256, "gate": False, "ragged": True, "reverse": True},
        {"name": "train_frames_bf16", "kind": "train", "dtype": "bf16", "B": 32, "T": 800, "H": 512, "gate": True, "ragged": True, "reverse": False},
        {"name": "train_long_f16", "kind": "train", "dtype": "f16", "B": 2, "T": 32769, "H": 1001, "gate": True, "ragged": False, "reverse": False},
        # one new token: a single stream, and a full serving batch of which some rows are idle
        {"name": "step_one_f32", "kind": "step", "dtype": "f32", "B": 1, "H": 1024, "gate": True, "idle": False},
        {"name": "step_batch_bf16", "kind": "step", "dtype": "bf16", "B": 64, "H": 2048, "gate": True, "idle": True},
        # optimizer steps: a small model, one of this package's size, the same in 8 bits with bf16 gradients, and a large
        # one with fp32 parameters, bf16 gradients and the bf16 copies the next forward pass reads
        {"name": "adamw32_small", "kind": "adamw", "bits": 32, "layers": 2, "width": 256, "param": "f32", "grad": "f32", "copy": ""},
        {"name": "adamw32_model", "kind": "adamw", "bits": 32, "layers": 8, "width": 512, "param": "f32", "grad": "f32", "copy": ""},
        {"name": "adamw8_model", "kind": "adamw", "bits": 8, "layers": 8, "width": 512, "param": "bf16", "grad": "bf16", "copy": ""},
        {"name": "adamw8_large", "kind": "adamw", "bits": 8, "layers": 20, "width": 1024, "param": "f32", "grad": "bf16", "copy": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "train", "step", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "step":
        return {"kind": kind, "dtype": dtype, "B": _log_int(rng, 1, 64), "H": _log_int(rng, 64, 2048), "gate": rng.random() < 0.6, "idle": rng.random() < 0.4}
    if kind == "adamw":
        param = rng.choice(["f32", "f32", "bf16", "f16"])
        return {"kind": kind, "bits": rng.choice([32, 8]), "layers": rng.randint(1, 12), "width": _log_int(rng, 48, 800), "param": param,
                "grad": rng.choice(["f32", "bf16", "f16"]), "copy": rng.choice(["", "bf16", "f16"]) if param == "f32" else ""}
    T, H = _log_int(rng, 2, 40000), _log_int(rng, 32, 1200)
    B = _log_int(rng, 1, max(1, min(64, 30_000_000 // (T * H))))
    return {"kind": kind, "dtype": dtype, "B": B, "T": T, "H": H, "gate": rng.random() < 0.6, "ragged": rng.random() < 0.5, "reverse": rng.random() < 0.4}


def _sizes(case):
    """The variables of a recurrent model of `layers` layers: an embedding, then for each layer a cell kernel, a convolution,
    and their biases, scales and offsets."""
    w = case["width"]
    sizes = [256 * w]
    for _ in range(case["layers"]):
        sizes += [2 * w * 4 * w, 4 * w, 5 * w * w, w, w]
    return sizes


def _offsets(sizes):
    off, at = [], 0
    for s in sizes:
        off.append(at)
        at += -(-s // BLOCK) * BLOCK
    return off, at


# ---- inputs --------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "adamw":
        return _prepare_adamw(case, gen)
    dt = DTYPES[case["dtype"]]
    B, T, H = case["B"], case.get("T", 1), case["H"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    # gates from mostly forgetting to a memory of about a thousand positions, by channel
    bias = torch.rand((H,), generator=gen, device="cuda") * 8.0 - 1.0
    if case["kind"] == "step":
        s = {"z": normal(B, H).to(dt), "f": (normal(B, H) + bias).to(dt), "o": normal(B, H).to(dt) if case["gate"] else None,
             "state": normal(B, H), "active": None}
        if case["idle"]:
            s["active"] = torch.rand((B,), generator=gen, device="cuda") < 0.75
    else:
        s = {"z": normal(B, T, H).to(dt), "f": (normal(B, T, H) + bias).to(dt), "o": normal(B, T, H).to(dt) if case["gate"] else None,
             "state": normal(B, H), "lens": None, "reverse": case["reverse"]}
        if case["ragged"]:
            s["lens"] = torch.randint(T // 2, T + 1, (B,), generator=gen, device="cuda")
        if case["kind"] == "train":
            s["dy"], s["dfinal"] = normal(B, T, H).to(dt), normal(B, H)
    s["kind"] = case["kind"]
    return s


def _prepare_adamw(case, gen):
    sizes = _sizes(case)
    off, total = _offsets(sizes)
    p = torch.zeros(total, dtype=DTYPES[case["param"]], device="cuda")
    g = torch.zeros(total, dtype=DTYPES[case["grad"]], device="cuda")
    m, r = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for i, (o, n) in enumerate(zip(off, sizes)):
        sigma = 10.0 ** (-2.0 - (i % 5) * 0.5)                 # gradients of different variables differ by orders of magnitude
        p[o:o + n] = (torch.randn(n, generator=gen, device="cuda") * 0.05).to(p.dtype)
        g[o:o + n] = (torch.randn(n, generator=gen, device="cuda") * sigma).to(g.dtype)
        m[o:o + n] = torch.randn(n, generator=gen, device="cuda") * (0.3 * sigma)
        r[o:o + n] = torch.exp(torch.randn(n, generator=gen, device="cuda") * 0.5) * sigma
    unseen = sizes[0] // 4                                      # embedding rows of symbols that have not occurred yet
    g[:unseen], m[:unseen], r[:unseen] = 0, 0, 0
    copy = torch.zeros(total, dtype=DTYPES[case["copy"]], device="cuda") if case["copy"] else None
    decay = [0.01 if n > 4 * case["width"] else 0.0 for n in sizes]
    s = {"kind": "adamw", "bits": case["bits"], "sizes": sizes, "off": off, "decay": decay, "p": p, "g": g, "copy": copy, "step": ADAM["step"]}
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _nearest8(m)
        s["v"], s["v_scale"] = _nearest8(r)
    else:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, r * r, None, None
    if own:
        from tacotron2_amd.training import AdamW
        views = lambda t: None if t is None else [t[o:o + n] for o, n in zip(off, sizes)]  # noqa: E731
        opt = AdamW(None, sizes, learning_rate=ADAM["lr"], beta1=ADAM["b1"], beta2=ADAM["b2"], epsilon=ADAM["eps"], weight_decay=decay,
                    state_bits=case["bits"], seed=ADAM["seed"])
        opt.load_state(s["m"], s["v"], ADAM["step"], m_scale=s["m_scale"], v_scale=s["v_scale"])
        s["opt"], s["bound"] = opt, opt.bind(views(g), views(p), copies=views(copy))
        s["m"], s["v"], s["m_scale"], s["v_scale"] = opt.m, opt.v, opt.m_scale, opt.v_scale
    return s


def _nearest8(x):
    """States that an earlier step left: e4m3 values and the power of two of each block."""
    b = x.view(-1, BLOCK)
    e = ((b.abs().amax(1).view(torch.int32) >> 23) - 7).clamp(min=16)
    q = torch.ldexp(b, (127 - e).view(-1, 1)).to(torch.float8_e4m3fn)
    return q.view(-1), e.to(torch.uint8).view(torch.float8_e8m0fnu)


# ---- one pass ------------------------------------------------------------------------------------------------------------
def run(s):
    return {"scan": _run_scan, "train": _run_train, "step": _run_step, "adamw": _run_adamw}[s["kind"]](s)


def _run_scan(s):
    if own:
        from tacotron2_amd import recurrence
        y, final = recurrence.gated_scan(None, s["z"], s["f"], s["o"], lens=s["lens"], state=s["state"], reverse=s["reverse"])
        return {"y": y, "final": final}
    x = _plain_forward(s)
    return {"y": x["y"].to(s["z"].dtype), "final": x["final"]}


def _run_train(s):
    if own:
        from tacotron2_amd import recurrence
        y, final, tape = recurrence.gated_scan(None, s["z"], s["f"], s["o"], lens=s["lens"], state=s["state"], reverse=s["reverse"], tape=True)
        dz, df, do, dstate = recurrence.gated_scan_backward(None, tape, s["dy"], s["dfinal"])
        return {"y": y, "final": final, "dz": dz, "df": df, "do": do, "dstate": dstate}
    dt = s["z"].dtype
    x = _plain_forward(s)
    turn = (lambda t: t.flip(1)) if s["reverse"] else (lambda t: t)
    dy = turn(s["dy"].float())
    dy = dy if x["live"] is None else torch.where(x["live"], dy, 0.0)
    d = dy if x["so"] is None else dy * x["so"]
    d = torch.cat([d[:, :-1], d[:, -1:] + s["dfinal"][:, None]], 1)
    # the gradient of h_t is d_t plus a_{t+1} times that of h_{t+1}: the same scan from the other end
    shifted = torch.cat([x["a"][:, 1:], torch.zeros_like(x["a"][:, :1])], 1)
    d = _doubling(shifted.flip(1), d.flip(1)).flip(1)
    before = torch.cat([s["state"][:, None], x["h"][:, :-1]], 1)
    out = {"y": x["y"].to(dt), "final": x["final"], "dstate": x["a"][:, 0] * d[:, 0]}
    dz, df = d * x["b"], d * (before - x["z"]) * x["a"] * x["b"]
    do = None if x["so"] is None else dy * x["h"] * x["so"] * (1.0 - x["so"])
    for name, t in (("dz", dz), ("df", df), ("do", do)):
        if t is not None and x["live"] is not None:
            t = torch.where(x["live"], t, 0.0)
        out[name] = None if t is None else turn(t).to(dt)
    return out


def _plain_forward(s):
    """h for all positions in the order of the recurrence, by doubling: after k rounds every position holds the composition of
    the last 2^k steps."""
    turn = (lambda t: t.flip(1)) if s["reverse"] else (lambda t: t)
    z, f = turn(s["z"].float()), turn(s["f"].float())
    a, b = torch.sigmoid(f), torch.sigmoid(-f)
    x = b * z
    live = None
    if s["lens"] is not None:
        live = turn(torch.arange(z.shape[1], device=z.device)[None, :, None] < s["lens"][:, None, None])
        a, b, x = torch.where(live, a, 1.0), torch.where(live, b, 0.0), torch.where(live, x, 0.0)
    x = torch.cat([x[:, :1] + a[:, :1] * s["state"][:, None], x[:, 1:]], 1)
    h = _doubling(a, x)
    so = None if s["o"] is None else torch.sigmoid(turn(s["o"].float()))
    y = h if so is None else h * so
    y = y if live is None else torch.where(live, y, 0.0)
    return {"z": z, "a": a, "b": b, "h": h, "so": so, "live": live, "y": turn(y), "final": h[:, -1].clone()}


def _doubling(a, x):
    d, T = 1, a.shape[1]
    while d < T:
        x = torch.cat([x[:, :d], torch.addcmul(x[:, d:], a[:, d:], x[:, :-d])], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return x


def _run_step(s):
    if own:
        from tacotron2_amd import recurrence
        y = recurrence.gated_scan_step(None, s["z"], s["f"], s["o"], s["state"], active=s["active"])
        return {"y": y, "state": s["state"]}
    z, f = s["z"].float(), s["f"].float()
    h = torch.sigmoid(f) * s["state"] + torch.sigmoid(-f) * z
    y = h if s["o"] is None else h * torch.sigmoid(s["o"].float())
    if s["active"] is not None:
        on = s["active"][:, None]
        h, y = torch.where(on, h, s["state"]), torch.where(on, y, 0.0)
    s["state"].copy_(h)
    return {"y": y.to(s["z"].dtype), "state": s["state"]}


def _run_adamw(s):
    keys = ("p", "m", "v") + (("m_scale", "v_scale") if s["bits"] == 8 else ()) + (("copy",) if s["copy"] is not None else ())
    if own:
        s["opt"].apply_gradients(s["bound"], clip_norm=ADAM["clip"])
        return {k: s[k] for k in keys}
    A = ADAM
    s["step"] += 1
    t = s["step"]
    norm = s["g"].double().square().sum().sqrt()
    g = s["g"].float() * (A["clip"] / norm.clamp(min=A["clip"])).float()
    padded = [-(-n // BLOCK) * BLOCK for n in s["sizes"]]
    keep = torch.tensor([1.0 - A["lr"] * w for w in s["decay"]], device=g.device).repeat_interleave(torch.tensor(padded, device=g.device))
    if s["bits"] == 8:
        m = _decode8(s["m"], s["m_scale"])
        r = _decode8(s["v"], s["v_scale"])
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * A["b1"] + g * (1.0 - A["b1"])
    v = v * A["b2"] + g * g * (1.0 - A["b2"])
    r = v.sqrt()
    p = s["p"].float() * keep - (A["lr"] / (1.0 - A["b1"] ** t)) * m / (r * (1.0 / math.sqrt(1.0 - A["b2"] ** t)) + A["eps"])
    s["p"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if s["bits"] == 8:
        word = _word(A["seed"], t, torch.arange(m.numel(), device=m.device))
        s["m"], s["m_scale"] = _encode8(m, word & 0xFFFF, False)
        s["v"], s["v_scale"] = _encode8(r, word >> 16, True)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return {k: s[k] for k in keys}


def _decode8(q, scale):
    return (q.float().view(-1, BLOCK) * scale.float().view(-1, 1)).view(-1)


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _word(seed, t, i):
    """32 bits for element i of step t."""
    h = _mix((seed ^ (20 * 0x9E3779B9)) & 0xFFFFFFFF)
    h = _mix(h ^ ((t * 0x85EBCA6B + 0x165667B1) & 0xFFFFFFFF))
    h = _mix(h ^ (((i >> 32) * 0xC2B2AE35 + 0x27D4EB2F) & 0xFFFFFFFF))
    return _mix(h ^ (((i & 0xFFFFFFFF) * 0x9E3779B1 + 0x85EBCA77) & 0xFFFFFFFF))


def _encode8(x, word16, keep_positive):
    """e4m3 codes of x over its block's power of two (the block's largest value lands in [128, 256)), rounded up with the
    probability that the cut-off part has."""
    b = x.view(-1, BLOCK)
    e = ((b.abs().amax(1).view(torch.int32) >> 23) - 7).clamp(min=16)
    # shifted so that a code is the upper bits of an fp32 number whose exponent field is the code's
    y = torch.ldexp(b.double(), (7 - e).view(-1, 1)).float().abs().view(torch.int32).view(-1)
    code = (y + (word16.to(torch.int32) << 4) + 8) >> 20
    if keep_positive:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = code | ((x.view(torch.int32) >> 24) & 0x80)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), e.to(torch.uint8).view(torch.float8_e8m0fnu)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "": 0}
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        state = 8 if case["bits"] == 32 else 2 + 2 / BLOCK
        return {"bytes": n * (2 * size[case["param"]] + size[case["grad"]] + 2 * state + size[case["copy"]]), "flops": 15.0 * n}
    gate = 1 if case["gate"] else 0
    es = size[case["dtype"]]
    if case["kind"] == "step":
        n = case["B"] * case["H"]
        return {"bytes": n * (es * (3 + gate) + 8), "flops": 12.0 * n}
    n = case["B"] * case["T"] * case["H"]
    live = 0.75 * n if case["ragged"] else n
    edge = 8 * case["B"] * case["H"]
    if case["kind"] == "scan":
        return {"bytes": es * (live * (2 + gate) + n) + edge, "flops": 12.0 * live}
    return {"bytes": es * (live * (3 + gate) + n * (3 + gate)) + 2 * edge, "flops": 37.0 * live}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "adamw":
        return _exact_adamw(case, seed)
    s = _inputs(case, seed)
    z, f = s["z"].double(), s["f"].double()
    so = None if s["o"] is None else 1.0 / (1.0 + torch.exp(-s["o"].double()))
    a, keep = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
    if case["kind"] == "step":
        h = a * s["state"].double() + keep * z
        y = h if so is None else so * h
        if s["active"] is not None:
            on = s["active"][:, None]
            h, y = torch.where(on, h, s["state"].double()), torch.where(on, y, 0.0)
        return {"y": y, "state": h}
    T = case["T"]
    lens = s["lens"]
    order = range(T - 1, -1, -1) if case["reverse"] else range(T)
    h = s["state"].double()
    hs, befores, on = torch.empty_like(z), torch.empty_like(z), None
    for t in order:
        befores[:, t] = h
        new = torch.addcmul(a[:, t] * h, keep[:, t], z[:, t])
        h = new if lens is None else torch.where((lens > t)[:, None], new, h)
        hs[:, t] = h
    y = hs if so is None else hs * so
    if lens is not None:
        on = (torch.arange(T, device=z.device)[None] < lens[:, None])[..., None]
        y = torch.where(on, y, 0.0)
    out = {"y": y, "final": h}
    if case["kind"] == "scan":
        return out
    dy = s["dy"].double()
    d = s["dfinal"].double()
    ds = torch.empty_like(z)
    for t in reversed(order):
        here = d + (dy[:, t] if so is None else dy[:, t] * so[:, t])
        ds[:, t] = here
        d = a[:, t] * here if lens is None else torch.where((lens > t)[:, None], a[:, t] * here, d)
    grads = {"dz": ds * keep, "df": ds * (befores - z) * a * keep, "do": None if so is None else dy * hs * so * (1.0 - so)}
    out.update({k: v if v is None or on is None else torch.where(on, v, 0.0) for k, v in grads.items()})
    return {**out, "dstate": d}


def _inputs(case, seed):
    """What prepare() makes, without the optimizer that a program keeps."""
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept


def _exact_adamw(case, seed):
    s = _inputs(case, seed)
    A, t = ADAM, ADAM["step"] + 1
    g = s["g"].double()
    g = g * min(1.0, A["clip"] / float(torch.linalg.vector_norm(g)))
    if case["bits"] == 8:
        m, r = (s[k].float().double().view(-1, BLOCK) * s[k + "_scale"].double()[:, None] for k in ("m", "v"))
        m, v = m.reshape(-1), (r * r).reshape(-1)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = A["b1"] * m + (1.0 - A["b1"]) * g
    v = A["b2"] * v + (1.0 - A["b2"]) * g * g
    p = s["p"].double()
    step = A["lr"] / (1.0 - A["b1"] ** t) * m / (torch.sqrt(v / (1.0 - A["b2"] ** t)) + A["eps"])
    for o, n, w in zip(s["off"], s["sizes"], s["decay"]):
        p[o:o + n] *= 1.0 - A["lr"] * w
    p = p - step
    out = {"p": p}
    if s["copy"] is not None:
        out["copy"] = p
    if case["bits"] == 32:
        return {**out, "m": m, "v": v}
    i = torch.arange(m.numel(), device=m.device)
    for key, x, shift in (("m", m, 0), ("v", torch.sqrt(v), 16)):
        top = x.abs().view(-1, BLOCK).amax(1)
        power = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=1e-300))), -200.0) - 7.0
        power = power.clamp(min=-111.0)
        u = x.abs().view(-1, BLOCK) / torch.exp2(power)[:, None]
        # the e4m3 step at u: an eighth of its power of two, 2^-9 below the normal range
        grid = torch.exp2(torch.floor(torch.log2(u.clamp(min=2.0 ** -6))) - 3.0)
        part = ((_word(A["seed"], t, i) >> shift) & 0xFFFF).double() / 65536.0 + 2.0 ** -17
        q = torch.floor(u / grid + part.view(-1, BLOCK)) * grid
        if shift:
            q = torch.where((x.view(-1, BLOCK) > 0) & (q == 0), 2.0 ** -9, q)
        out[key] = (torch.sign(x).view(-1, BLOCK) * q).view(-1)
        out[key + "_scale"] = torch.exp2(power)
    return out
