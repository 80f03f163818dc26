"""Cases of the optimizer-side operators over lists of tensors: the global gradient norm with its clip coefficient,
clipping in place, and the AdamW step.

A case lays out its tensors in one or two buffers, the way an allocator or a flat gradient buffer does; the buffers come
back whole, so that what lies between the tensors is compared too.  Every pass leaves the state ready for the next one:
clipping follows a bound that is lowered a little every pass (as a bound tied to a falling gradient norm is), so that each
pass does clip; the AdamW step counts its steps.
"""

import math
import random

import torch

own = False

GRAD_STD = 1e-3
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
NORMS = {"1": 1.0, "2": 2.0, "inf": math.inf}
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1
FIRST_STEP = 10
BOUND_DECAY = 0.9999


# ------------------------------------------------------------------------------------------------ cases ----
def listed():
    return [
        # the few parameters that a wrapped model keeps outside its sharded groups: nothing but latency
        {"name": "norm: 9 small fp32", "op": "norm", "norm": "2", "grad": "float32", "second": "", "layout": "spread",
         "tensors": 9, "low": 64, "high": 4096, "pick": 1, "spacing": 128},
        # the 16-bit gradients of one decoder layer as autograd leaves them
        {"name": "norm: a layer, bf16", "op": "norm", "norm": "2", "grad": "bfloat16", "second": "", "layout": "layer",
         "width": 4096, "inner": 14336, "narrow": 1024, "layers": 1, "spacing": 256},
        # a model of many odd tensors, part of its gradients in binary32, watched by its largest gradient
        {"name": "norm: 1427 ragged, inf", "op": "norm", "norm": "inf", "grad": "float32", "second": "bfloat16",
         "layout": "spread", "tensors": 1427, "low": 1, "high": 1048576, "pick": 2, "spacing": 8},
        # the same kind of watch with the 1-norm on half-precision gradients
        {"name": "norm: 300 fp16, 1-norm", "op": "norm", "norm": "1", "grad": "float16", "second": "", "layout": "spread",
         "tensors": 300, "low": 1000, "high": 2000000, "pick": 3, "spacing": 256},
        # biases and norm weights of a small model, clipped every step
        {"name": "clip: 48 small fp32", "op": "clip", "norm": "2", "grad": "float32", "second": "", "layout": "spread",
         "tensors": 48, "low": 64, "high": 4096, "pick": 4, "spacing": 128},
        # low-rank adapters of every projection of a model: many tensors of one size
        {"name": "clip: 448 adapters, bf16", "op": "clip", "norm": "2", "grad": "bfloat16", "second": "",
         "layout": "spread", "tensors": 448, "low": 65536, "high": 65536, "pick": 5, "spacing": 256},
        # one rank's binary32 gradient shard of a layer: nine fragments back to back, starting at odd places
        {"name": "clip: shard fragments, fp32", "op": "clip", "norm": "2", "grad": "float32", "second": "",
         "layout": "spread", "tensors": 9, "low": 500001, "high": 8000003, "pick": 6, "spacing": 1},
        # the 16-bit gradients of four decoder layers at once
        {"name": "clip: 4 layers, bf16", "op": "clip", "norm": "2", "grad": "bfloat16", "second": "", "layout": "layer",
         "width": 4096, "inner": 14336, "narrow": 1024, "layers": 4, "spacing": 256},
        # the norm weights of a 32-layer decoder, stepped outside any group
        {"name": "adamw: 65 norm weights", "op": "adamw", "grad": "float32", "second": "", "layout": "spread",
         "tensors": 65, "low": 4096, "high": 4096, "pick": 7, "spacing": 128},
        # masters of many odd tensors with 16-bit gradients and a 16-bit copy of the parameters
        {"name": "adamw: 573 ragged, bf16", "op": "adamw", "grad": "bfloat16", "second": "bfloat16", "layout": "spread",
         "tensors": 573, "low": 1, "high": 1048576, "pick": 8, "spacing": 8},
        # a whole decoder layer with binary32 gradients, scaled by the clip coefficient in the same pass
        {"name": "adamw: a layer, fp32", "op": "adamw", "grad": "float32", "second": "", "layout": "layer",
         "width": 4096, "inner": 14336, "narrow": 1024, "layers": 1, "spacing": 128},
        # the layer trained with 16-bit gradients: masters, moments and the 16-bit parameters of the next forward
        {"name": "adamw: a layer, bf16", "op": "adamw", "grad": "bfloat16", "second": "bfloat16", "layout": "layer",
         "width": 4096, "inner": 14336, "narrow": 1024, "layers": 1, "spacing": 256},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "adamw"])
    case = {"op": op, "grad": rng.choice(["float32", "bfloat16", "float16"]), "second": ""}
    if op == "adamw":
        case["second"] = rng.choice(["", "bfloat16", "float16"])  # the 16-bit copy of the parameters
        most = 100_000_000
    else:
        case["norm"] = rng.choice(["1", "2", "2", "inf"])
        case["second"] = rng.choice(["", "", "float32", "bfloat16"])  # every other tensor in another type
        if case["second"] == case["grad"]:
            case["second"] = ""
        most = 400_000_000
    if rng.random() < 0.25:
        width = 64 * _log_uniform(rng, 2, 64)
        layer = 2 * width * width + 2 * width * (width // 4) + 12 * width * width + 2 * width
        layers = rng.randint(1, max(1, min(8, most // layer)))
        case.update(layout="layer", width=width, inner=4 * width, narrow=width // 4, layers=layers)
    else:
        tensors = _log_uniform(rng, 1, 1500)
        mean = _log_uniform(rng, 100, max(101, most // tensors))
        high = min(most // tensors, 4 * mean)
        case.update(layout="spread", tensors=tensors, low=max(1, min(high, mean // rng.choice([1, 30, 1000]))), high=high,
                    pick=rng.randrange(1 << 30))
    case["spacing"] = rng.choice([1, 1, 8, 256])
    return case


def _numels(case):
    if case["layout"] == "layer":
        w, f, k = case["width"], case["inner"], case["narrow"]
        return [w * w, w * k, w * k, w * w, w * f, w * f, w * f, w, w] * case["layers"]
    rng = random.Random(case["pick"])
    return [_log_uniform(rng, case["low"], case["high"]) for _ in range(case["tensors"])]


def _places(numels, spacing):
    """Where each tensor starts in its buffer (elements), and the buffer's length.  ``spacing`` 1: back to back behind
    three elements of somebody else's; otherwise every tensor starts at a multiple of it, with a gap behind each."""
    at, starts = (3 if spacing == 1 else 0), []
    for n in numels:
        starts.append(at)
        at += n
        if spacing > 1:
            at = (at // spacing + 1) * spacing
    return starts, at + 5


def _buffer(numels, spacing, dtype, gen, std):
    starts, total = _places(numels, spacing)
    buf = torch.empty(total, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)
    return buf, [buf[s:s + n] for s, n in zip(starts, numels)]


# ---------------------------------------------------------------------------------------------- prepare ----
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    numels = _numels(case)
    dtype = DTYPES[case["grad"]]
    state = {"op": case["op"]}
    if case["op"] == "adamw":
        spacing = case["spacing"]
        p_buf, state["params"] = _buffer(numels, spacing, torch.float32, gen, 0.02)
        g_buf, state["grads"] = _buffer(numels, spacing, dtype, gen, GRAD_STD)
        m_buf, state["exp_avgs"] = _buffer(numels, spacing, torch.float32, gen, GRAD_STD)
        v_buf, state["exp_avg_sqs"] = _buffer(numels, spacing, torch.float32, gen, GRAD_STD)
        v_buf.square_()
        state["buffers"] = [p_buf, m_buf, v_buf]
        state["outs16"] = None
        if case["second"]:
            o_buf, state["outs16"] = _buffer(numels, spacing, DTYPES[case["second"]], gen, 0.02)
            state["buffers"].append(o_buf)
        state["grad_scale"] = torch.full((1,), 0.75, device="cuda")
        state["step"] = FIRST_STEP
        return state
    if case["second"]:
        a_buf, a = _buffer(numels[0::2], case["spacing"], dtype, gen, GRAD_STD)
        b_buf, b = _buffer(numels[1::2], case["spacing"], DTYPES[case["second"]], gen, GRAD_STD)
        grads = [(b if i % 2 else a)[i // 2] for i in range(len(numels))]
        state["buffers"] = [a_buf, b_buf]
    else:
        buf, grads = _buffer(numels, case["spacing"], dtype, gen, GRAD_STD)
        state["buffers"] = [buf]
    state["grads"] = grads
    state["norm_type"] = NORMS[case["norm"]]
    state["bound"] = _first_bound(case, sum(numels))
    return state


def _first_bound(case, n):
    """Well below the norm of ``n`` normal numbers."""
    return GRAD_STD * {"1": 0.3 * n, "2": 0.37 * math.sqrt(n), "inf": 0.9}[case["norm"]]


# -------------------------------------------------------------------------------------------------- run ----
def run(state):
    if state["op"] == "adamw":
        state["step"] += 1
        if own:
            from yafsdp_amd.optim import list_adamw_step

            list_adamw_step(state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"], state["outs16"],
                            step=state["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                            grad_scale=state["grad_scale"])
        else:
            _adamw(state)
        return {"buffers": state["buffers"]}
    if state["op"] == "norm":
        if own:
            from yafsdp_amd.optim import list_clip_coef

            norm, coef = list_clip_coef(state["grads"], state["bound"], state["norm_type"])
        else:
            norm = _norm(state["grads"], state["norm_type"])
            coef = _coef(norm, state["bound"])
        return {"norm": norm, "coef": coef}
    state["bound"] *= BOUND_DECAY
    if own:
        from yafsdp_amd.optim import list_clip_grad_norm_

        norm = list_clip_grad_norm_(state["grads"], state["bound"], state["norm_type"])
    else:
        norm = _norm(state["grads"], state["norm_type"])
        coef = _coef(norm, state["bound"])
        [g.copy_(g.float() * coef) for g in state["grads"]]
    return {"norm": norm, "buffers": state["buffers"]}


def _norm(grads, norm_type):
    if norm_type == math.inf:
        return torch.stack([g.abs().max().float() for g in grads]).max()
    if norm_type == 1.0:
        return torch.stack([g.float().abs().sum() for g in grads]).sum()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _coef(norm, bound):
    return torch.clamp(bound / (norm + 1e-6), max=1.0)


def _adamw(state):
    t = state["step"]
    step_size, root = LR / (1.0 - BETA1 ** t), math.sqrt(1.0 - BETA2 ** t)
    [_adamw_one(*tensors, state["grad_scale"], step_size, root)
     for tensors in zip(state["params"], state["grads"], state["exp_avgs"], state["exp_avg_sqs"])]
    if state["outs16"] is not None:
        [o.copy_(p) for o, p in zip(state["outs16"], state["params"])]


def _adamw_one(p, g, m, v, scale, step_size, root):
    g = g.float() * scale
    p.mul_(1.0 - LR * DECAY)
    m.add_((g - m) * (1.0 - BETA1))
    v.mul_(BETA2).add_((1.0 - BETA2) * g * g)
    p.sub_(step_size * m / (v.sqrt() / root + EPS))


# ----------------------------------------------------------------------------------------- work and exact ----
def work(case):
    numels = _numels(case)
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    n = sum(numels)
    if case["op"] == "adamw":
        per = 24 + size[case["grad"]] + (2 if case["second"] else 0)
        return {"bytes": per * n, "flops": 16 * n}
    read = sum(k * size[case["second"] if case["second"] and i % 2 else case["grad"]] for i, k in enumerate(numels))
    if case["op"] == "norm":
        return {"bytes": read + 8, "flops": 2 * n}
    return {"bytes": 2 * read + 8, "flops": 3 * n}


def exact(case, seed):
    state = prepare(case, seed)
    numels = _numels(case)
    if case["op"] == "adamw":
        starts, _ = _places(numels, case["spacing"])
        wide = [b.double() for b in state["buffers"][:3]]
        if case["second"]:
            wide.append(state["buffers"][3].double())
        t = FIRST_STEP + 1
        for s, n, g in zip(starts, numels, state["grads"]):
            p, m, v = (w.narrow(0, s, n) for w in wide[:3])
            g = 0.75 * g.double()
            m_new = BETA1 * m + (1.0 - BETA1) * g
            v_new = BETA2 * v + (1.0 - BETA2) * g ** 2
            m_hat, v_hat = m_new / (1.0 - BETA1 ** t), v_new / (1.0 - BETA2 ** t)
            p_new = p - LR * DECAY * p - LR * m_hat / (torch.sqrt(v_hat) + EPS)
            m.copy_(m_new), v.copy_(v_new), p.copy_(p_new)
            if case["second"]:
                wide[3].narrow(0, s, n).copy_(p_new)
        return {"buffers": wide}
    kind = case["norm"]
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in state["grads"]:
        a = torch.abs(g.double())
        if kind == "inf":
            total = torch.maximum(total, a.max())
        else:
            total = total + (a.sum() if kind == "1" else torch.dot(a, a))
    norm = torch.sqrt(total) if kind == "2" else total
    bound = _first_bound(case, sum(numels)) * (BOUND_DECAY if case["op"] == "clip" else 1.0)
    coef = torch.minimum(bound / (norm + 1e-6), torch.ones_like(norm))
    if case["op"] == "norm":
        return {"norm": norm, "coef": coef}
    wide = [b.double() for b in state["buffers"]]
    halves = [numels[0::2], numels[1::2]] if case["second"] else [numels]
    for w, part in zip(wide, halves):
        for s, n in zip(_places(part, case["spacing"])[0], part):
            w.narrow(0, s, n).mul_(coef)
    return {"norm": norm, "buffers": wide}
