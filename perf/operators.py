"""Cases of the many-tensor AdamW steps and of gradient norms: inputs, plain forms and the library's calls.

Three operators, each over a whole set of parameter tensors at once:

* ``adamw``: decoupled weight decay, moments in 32 bits, optionally 32-bit master weights beside 16-bit parameters;
* ``adamw8``: the same step with moments in 8 bits, and the moments it leaves as 32-bit numbers;
* ``norm`` and ``clip``: the 2-norm over all gradients, and scaling the gradients to a largest norm.

The tensors of a set are views of flat buffers, one buffer for each kind of tensor (with and without weight decay, moments
in 8 or in 32 bits), as a training program that exchanges its parameters in one collective keeps them. The plain forms work
on those buffers.
"""

import math
import random

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100
SMALLEST_8BIT = 4096   # tensors with fewer elements keep 32-bit moments
FLOOR = 2.0 ** -100    # smallest block scale

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------- cases


def listed():
    return [
        # a classifier head and its norm tuned alone: four tensors, 5 k elements, all latency
        dict(name="adamw_head_fp32", op="adamw", set="head", type="fp32"),
        # a small vision transformer trained in fp32: 102 tensors, two thirds of them vectors
        dict(name="adamw_vit14m_fp32", op="adamw", set="vit", type="fp32"),
        # a character language model in bf16 with fp32 master weights and clipping, the common training recipe
        dict(name="adamw_charlm40m_bf16_master", op="adamw", set="charlm", type="bf16", master=True, max_norm=1.0),
        # a 700M decoder in fp32: the largest step, bound by memory
        dict(name="adamw_decoder700m_fp32", op="adamw", set="decoder", type="fp32"),
        # odd sizes packed without gaps (no tensor aligned), fp16
        dict(name="adamw_odd_packed_fp16", op="adamw", set="random", tensors=57, numel=9_437_411, shapes=5, type="fp16", packed=True),
        # one weight matrix with 8-bit moments: the smallest call
        dict(name="adamw8_weight_fp32", op="adamw8", set="weight", type="fp32", block=128),
        # 8-bit moments for bf16 training, small vectors beside large matrices
        dict(name="adamw8_charlm40m_bf16", op="adamw8", set="charlm", type="bf16", block=128, max_norm=1.0),
        # 8-bit moments of a 700M decoder, bf16 parameters
        dict(name="adamw8_decoder700m_bf16", op="adamw8", set="decoder", type="bf16", block=256),
        # odd sizes: blocks that end inside, tensors shorter than a block
        dict(name="adamw8_odd_fp32", op="adamw8", set="random", tensors=31, numel=21_000_037, shapes=9, type="fp32", block=64),
        # the norm of a vision transformer's gradients, logged every step
        dict(name="norm_vit14m_fp32", op="norm", set="vit", type="fp32"),
        # the norm of a decoder's bf16 gradients
        dict(name="norm_decoder700m_bf16", op="norm", set="decoder", type="bf16"),
        # gradients clipped in place before a step that does not clip by itself
        dict(name="clip_charlm40m_fp32", op="clip", set="charlm", type="fp32", max_norm=1.0),
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm", "clip"])
    numel = int(math.exp(rng.uniform(math.log(2_000), math.log(150_000_000))))
    case = dict(op=op, set="random", tensors=rng.randint(1, 160), numel=numel, shapes=rng.randrange(1 << 20),
                type=rng.choice(["fp32", "bf16", "fp16"]))
    if op != "adamw8" and rng.random() < 0.25:
        case["packed"] = True
    if op == "adamw8":
        case["block"] = rng.choice([64, 128, 256])
    if op.startswith("adamw") and case["type"] != "fp32" and rng.random() < 0.5:
        case["master"] = True
    if op == "clip" or (op.startswith("adamw") and rng.random() < 0.4):
        case["max_norm"] = rng.choice([0.25, 1.0, 4.0])
    return case


def _blocks(width, depth, hidden):
    one = [(width,), (width,), (width, 3 * width), (3 * width,), (width, width), (width,),
           (width,), (width,), (width, hidden), (hidden,), (hidden, width), (width,)]
    return one * depth


def _shapes(case):
    kind = case["set"]
    if kind == "head":
        return [(384,), (384,), (384, 10), (10,)]
    if kind == "weight":
        return [(1024, 1024)]
    if kind == "vit":
        return [(192, 384), (384,)] + _blocks(384, 8, 1536) + [(384,), (384,), (384, 10), (10,)]
    if kind == "charlm":
        return [(256, 512)] + _blocks(512, 12, 2048) + [(512,), (512,), (512, 256)]
    if kind == "decoder":
        return [(1536, 4608), (1536, 1536), (1536, 6144), (6144, 1536)] * 24 + [(50304, 1536)]
    r = random.Random(case["shapes"])
    parts = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    sizes = [(max(1, int(case["numel"] * x / sum(parts))), r.choice([1, 1, 3, 8, 17])) for x in parts]
    return [(rows, n // rows) if rows > 1 and n >= 64 * rows else (n,) for n, rows in sizes]


def _numel(shape):
    return math.prod(shape)


def _segments(case):
    """The flat buffers of a case: [(decay, eight bits?, [(offset, shape)], length)]."""
    packed, groups = case.get("packed", False), {}
    for shape in _shapes(case):
        decay = DECAY if len(shape) > 1 else 0.0
        eight = case["op"] == "adamw8" and _numel(shape) >= SMALLEST_8BIT
        views, length = groups.get((decay, eight), ([], 0))
        groups[decay, eight] = views + [(length, shape)], length + (_numel(shape) if packed else -(-_numel(shape) // 256) * 256)
    return [(d, e, views, length) for (d, e), (views, length) in sorted(groups.items())]


def work(case):
    e, op = _SIZES[case["type"]], case["op"]
    if op == "norm":
        n = sum(_numel(s) for s in _shapes(case))
        return {"bytes": e * n + 4, "flops": 2 * n}
    if op == "clip":
        n = sum(_numel(s) for s in _shapes(case))
        return {"bytes": 2 * e * n + 4, "flops": 3 * n}
    bytes_, flops = 0, 0
    for _, eight, views, _ in _segments(case):
        n = sum(_numel(s) for _, s in views)
        # parameter and gradient; a master copy is read and written, the parameter then only written
        bytes_ += n * ((2 * e + 8) if case.get("master") else 3 * e)
        if eight:
            # codes and scales read and written, the moments written as 32-bit numbers
            blocks = sum(-(-_numel(s) // case["block"]) for _, s in views)
            bytes_ += 4 * n + 16 * blocks + 8 * n
            flops += 32 * n
        else:
            bytes_ += 16 * n
            flops += 14 * n
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------- inputs


def _random(n, views, gen, scale, spread):
    """N(0, scale) whose size varies from stretch to stretch of 1024 elements; zero between the views."""
    x = torch.randn(n, device="cuda", generator=gen).mul_(scale)
    if spread:
        k = -(-n // 1024)
        size = torch.randn(k, device="cuda", generator=gen).mul_(spread).exp_()
        x.mul_(size.repeat_interleave(1024)[:n])
    ends = [o + _numel(s) for o, s in views]
    [x[end:begin].zero_() for end, begin in zip(ends, [o for o, _ in views[1:]] + [n])]
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, op = _TYPES[case["type"]], case["op"]
    state = {"case": case, "step": STEP, "segments": []}
    for decay, eight, views, n in _segments(case):
        seg = {"decay": decay, "eight": eight, "views": views}
        # gradients with stretches of zeros (rows of an embedding that no token used)
        live = (torch.rand(-(-n // 1024), device="cuda", generator=gen) > 1 / 16).float()
        g = _random(n, views, gen, 1e-3, 0.7).mul_(live.repeat_interleave(1024)[:n])
        seg["g"] = g.to(kind)
        if op.startswith("adamw"):
            p = _random(n, views, gen, 0.02, 0.0)
            seg["p"] = p.to(kind)
            if case.get("master"):
                seg["master"] = p
            m = _random(n, views, gen, 3e-4, 0.7)
            v = _random(n, views, gen, 1e-3, 0.7).square_().add_(m.square())
            if eight:
                seg["m_q"], seg["m_s"], seg["v_q"], seg["v_s"] = _encode(m, v.sqrt_(), case["block"])
                m.zero_()
                v.zero_()
            seg["m"], seg["v"] = m, v
        state["segments"].append(seg)
    if own:
        import smo_optimizer_b200 as smo

        groups, states, out = [], [], []
        for seg in state["segments"]:
            params = []
            for o, shape in seg["views"]:
                n = _numel(shape)
                p = torch.nn.Parameter((seg["p"] if "p" in seg else seg["g"])[o:o + n].view(shape))
                p.grad = seg["g"][o:o + n].view(shape)
                params.append(p)
                st = {"step": STEP}
                if "p" not in seg:
                    continue
                if seg["eight"]:
                    b = case["block"]
                    first, last = o // b, o // b + -(-n // b)
                    st.update({k: seg[k][first:last] for k in ("m_q", "m_s", "v_q", "v_s")})
                    out.append((seg["m"][o:o + n].view(shape), seg["v"][o:o + n].view(shape)))
                else:
                    st.update(exp_avg=seg["m"][o:o + n].view(shape), exp_avg_sq=seg["v"][o:o + n].view(shape))
                if "master" in seg:
                    st["master"] = seg["master"][o:o + n].view(shape)
                states.append((p, st))
            groups.append({"params": params, "weight_decay": seg["decay"]})
        state["params"] = [p for g in groups for p in g["params"]]
        if states:
            kw = dict(lr=LR, betas=(BETA1, BETA2), eps=EPS, master_weights=bool(case.get("master")), max_grad_norm=case.get("max_norm"))
            if case["op"] == "adamw8":
                opt = smo.AdamW8bit(groups, block_size=case["block"], min_8bit_numel=SMALLEST_8BIT, **kw)
                state["eight"] = [p for g, seg in zip(groups, state["segments"]) if seg["eight"] for p in g["params"]]
                state["out"] = out
            else:
                opt = smo.AdamW(groups, **kw)
            for p, st in states:
                opt.state[p] = st
            state["opt"] = opt
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    segs = state["segments"]
    if case["op"] in ("norm", "clip"):
        norm = _norm(segs)
        if case["op"] == "norm":
            return {"norm": norm}
        c = _coefficient(norm, case["max_norm"])
        return {"norm": norm, "g": [s["g"].copy_(s["g"].float() * c) for s in segs]}
    state["step"] += 1
    norm = _norm(segs) if case.get("max_norm") else None
    c = _coefficient(norm, case["max_norm"]) if case.get("max_norm") else None
    return _outputs(case, [_step(case, state, s, c) for s in segs], norm)


def _run_own(case, state):
    import smo_optimizer_b200 as smo

    if case["op"] == "norm":
        return {"norm": smo.grad_norm(state["params"])}
    if case["op"] == "clip":
        return {"norm": smo.clip_grad_norm_(state["params"], case["max_norm"]), "g": [s["g"] for s in state["segments"]]}
    opt = state["opt"]
    opt.step()
    if case["op"] == "adamw8" and state["eight"]:
        opt.moments(state["eight"], out=state["out"])
    return _outputs(case, state["segments"], opt.last_grad_norm if case.get("max_norm") else None)


def _outputs(case, segs, norm):
    got = {k: [s[k] for s in segs] for k in ("p", "m", "v") + (("master",) if case.get("master") else ())}
    return got if norm is None else dict(got, norm=norm)


def _norm(segs):
    return torch.stack([s["g"].double().square().sum() for s in segs]).sum().sqrt().float()


def _coefficient(norm, max_norm):
    return (torch.full_like(norm, max_norm) / (norm + 1e-6)).clamp(max=1.0)


def _decode(q, s, top):
    """Codes of `top` steps as the 32-bit numbers they stand for: s (q / top)^2 with q's sign."""
    q = q.float()
    return q * q.abs() * (s * (1.0 / (top * top)))


def _codes(x, top):
    s = x.abs().amax(1, keepdim=True).clamp(min=FLOOR)
    q = ((x.abs() * torch.reciprocal(s)).clamp(min=FLOOR).sqrt() * float(top)).round().nan_to_num(0.0)
    return q, s


def _encode(m, u, block):
    m, u = m.view(-1, block), u.view(-1, block)
    qm, sm = _codes(m, 127)
    qu, su = _codes(u, 255)
    qu = torch.where((u > 0) & (qu == 0), 1.0, qu)
    return torch.copysign(qm, m).to(torch.int8), sm, qu.to(torch.uint8), su


def _step(case, state, seg, c):
    g = seg["g"].float()
    if c is not None:
        g = g * c
    if seg["eight"]:
        m, u = _decode(seg["m_q"], seg["m_s"], 127).view(-1), _decode(seg["v_q"], seg["v_s"], 255).view(-1)
        v = u.square_()
    else:
        m, v = seg["m"], seg["v"]
    m.mul_(BETA1).add_(g * (1 - BETA1))
    v.mul_(BETA2).add_(g * (1 - BETA2) * g)
    root = v.sqrt()
    t = state["step"]
    held = seg["master"] if "master" in seg else seg["p"].float()
    update = (m * (LR / (1 - BETA1 ** t))).div_((root * (1 / math.sqrt(1 - BETA2 ** t))).add_(EPS))
    held.mul_(1 - LR * seg["decay"]).sub_(update)
    if held is not seg["p"]:
        seg["p"].copy_(held)
    if seg["eight"]:
        codes = _encode(m, root, case["block"])
        seg["m_q"].copy_(codes[0]), seg["m_s"].copy_(codes[1]), seg["v_q"].copy_(codes[2]), seg["v_s"].copy_(codes[3])
        seg["m"].copy_(_decode(seg["m_q"], seg["m_s"], 127).view(-1))
        seg["v"].copy_(_decode(seg["v_q"], seg["v_s"], 255).view(-1).square_())
    return seg


# ---------------------------------------------------------------- the definition in 64 bits


def _r32(x):
    """The nearest 32-bit number: where the definition holds a number in 32 bits."""
    return x.to(torch.float32).to(torch.float64)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    segs, op = state["segments"], case["op"]
    total = sum(float(torch.linalg.vector_norm(x.double())) ** 2 for s in segs for x in s["g"].split(1 << 26))
    norm = math.sqrt(total)
    if op == "norm":
        return {"norm": torch.tensor(norm, dtype=torch.float64)}
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float64).to(torch.float32))  # noqa: E731

    def moments_8bit(s, a, e, g, pieces):
        """Moments of elements a..e with codes decided on 32-bit numbers: every operation in 64 bits, rounded once."""
        b = case["block"]
        rows = slice(a // b, -(-e // b))
        cm, cu = s["m_q"][rows].double(), s["v_q"][rows].double()
        m = _r32(torch.sign(cm) * cm * cm * _r32(s["m_s"][rows].double() * f32(1 / 16129))).view(-1)
        u = _r32(cu * cu * _r32(s["v_s"][rows].double() * f32(1 / 65025))).view(-1)
        m = _r32(_r32(m * f32(BETA1)) + _r32(g * f32(1 - BETA1)))
        v = _r32(_r32(_r32(u * u) * f32(BETA2)) + _r32(_r32(g * f32(1 - BETA2)) * g))
        u = _r32(torch.sqrt(v))
        for key, x, top in (("m", m, 127), ("v", u, 255)):
            x = x.view(-1, b)
            scale = torch.clamp(x.abs().max(dim=1, keepdim=True).values, min=FLOOR)
            q = torch.round(_r32(top * _r32(torch.sqrt(_r32(x.abs() * _r32(1 / scale))))))
            if key == "v":
                q = torch.maximum(q, (x > 0).double())
            held = (torch.sign(x) * q * q * scale / (top * top)).view(-1)
            pieces[key].append(held if key == "m" else held * held)
        return m, v

    c = None
    if case.get("max_norm"):
        c = min(1.0, f32(case["max_norm"] / f32(f32(norm) + f32(1e-6))))
    if op == "clip":
        return {"norm": torch.tensor(norm, dtype=torch.float64), "g": [s["g"].double() * c for s in segs]}
    got = {"p": [], "m": [], "v": [], "master": []}
    t = STEP + 1
    size = LR / (1 - BETA1 ** t)
    root2 = math.sqrt(1 - BETA2 ** t)
    for s in segs:
        pieces = {k: [] for k in got}
        n, piece = s["g"].numel(), 1 << 26
        for a in range(0, n, piece):
            e = min(n, a + piece)
            g = s["g"][a:e].double() * (1.0 if c is None else c)
            p = (s["master"] if "master" in s else s["p"])[a:e].double()
            if s["eight"]:
                m, v = moments_8bit(s, a, e, _r32(g), pieces)
            else:
                m = BETA1 * s["m"][a:e].double() + (1 - BETA1) * g
                v = BETA2 * s["v"][a:e].double() + (1 - BETA2) * g * g
                pieces["m"].append(m)
                pieces["v"].append(v)
            p = p * (1 - LR * s["decay"]) - size * m / (torch.sqrt(v) / root2 + EPS)
            pieces["p"].append(p)
        for k in ("p", "m", "v"):
            got[k].append(torch.cat(pieces[k]))
        if "master" in s:
            got["master"].append(got["p"][-1])
        s.clear()
    if not got["master"]:
        del got["master"]
    if c is not None:
        got["norm"] = torch.tensor(norm, dtype=torch.float64)
    return got
