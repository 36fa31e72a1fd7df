"""Cases that measure the operators over many tensors at once (`pde_surrogate_amd.optim`): the AdamW step with 32-bit or
8-bit states, with or without clipping by the gradients' common norm, and the clipping alone.

A program keeps its parameters and gradients as views of flat buffers; every tensor begins at a multiple of 256 elements, as
separate allocations do, and what lies between two tensors is zero.  The plain form computes on the flat buffers.

    `own` False   elementary torch operations in 32 bits (the norm's sum in 64), rounded once at the end
    `own` True    optim.FusedAdamW.step() and optim.clip_grad_norm_()

8-bit states: blocks of 256 elements of one tensor (the last one may be partly filled) share a 32-bit scale, and both the
first moment m and the root r of the second are held as e4m3 numbers with stochastic rounding: the value x / scale is
rounded down after a number from [0, 1) steps of its binade has been added.  That number comes from the seed, the step, the
tensor's place in the list, the block and the place in it (`dither`), so equal inputs give equal states.
"""
import math
import random

import torch

own = False

BLOCK = 256
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, BETA1, EPS, DECAY, SEED = 3e-4, 0.9, 1e-8, 0.1, 1234
TOP, TINY = 448.0, 2.0 ** -100         # the largest e4m3 number; a block whose largest value is under TINY is held as zeros
GOLD, MIX_A, MIX_B = 0x9E3779B9, 0x6A09E667, 0xBB67AE85     # fractions of the golden ratio, sqrt 2 and sqrt 3; odd


# ---- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    def case(name, op, set, dtype="float32", bits=32, master=False, clip=False, beta2=0.999, **sizes):
        return dict(name=name, op=op, set=set, dtype=dtype, bits=bits, master=master, clip=clip, beta2=beta2, **sizes)
    return [
        # one small vector (a norm's weight trained alone): the call's latency
        case("step32 one vector", "step", "ragged", count=1, elements=1003, sizes=1),
        # the default DenseED's 82 parameters, as its training loop steps them
        case("step32 densed", "step", "densed"),
        # a ragged list of a few hundred tensors, clipped: the conditional flow's many small layers at a larger width
        case("step32 ragged clipped", "step", "ragged", clip=True, count=300, elements=20000003, sizes=2),
        # bf16 weights whose low halves are kept: the usual mixed-precision training of a transformer
        case("step32 bf16 master stack", "step", "stack", "bfloat16", master=True, beta2=0.95, hidden=2048, layers=3, vocab=32000),
        # the largest: float32 weights
        case("step32 large stack", "step", "stack", beta2=0.95, hidden=4096, layers=1, vocab=32000),
        # the same lists with 8-bit states
        case("step8 densed", "step", "densed", bits=8),
        case("step8 ragged clipped", "step", "ragged", bits=8, clip=True, count=61, elements=3000017, sizes=3),
        case("step8 bf16 master clipped", "step", "stack", "bfloat16", bits=8, master=True, clip=True, beta2=0.95, hidden=1024,
             layers=8, vocab=50257),
        case("step8 bf16 large stack", "step", "stack", "bfloat16", bits=8, beta2=0.95, hidden=4096, layers=1, vocab=32000),
        # clipping in a training that is under its limit, as most steps are: the norm is found and no gradient changes
        case("clip densed", "clip", "densed"),
        case("clip fp16 ragged", "clip", "ragged", "float16", count=130, elements=9000001, sizes=4),
        case("clip bf16 large stack", "clip", "stack", "bfloat16", hidden=4096, layers=1, vocab=32000),
    ]


def draw(rng):
    op = rng.choice(("step", "step", "step", "step", "clip"))
    dtype = rng.choice(("float32", "float32", "bfloat16", "bfloat16", "float16"))
    c = dict(op=op, dtype=dtype, bits=rng.choice((32, 8)) if op == "step" else 32, master=False, clip=False, beta2=rng.choice((0.95, 0.99, 0.999)))
    if op == "step":
        c["master"] = dtype == "bfloat16" and rng.random() < 0.5
        c["clip"] = rng.random() < 0.4
    c["set"] = rng.choice(("ragged", "ragged", "stack", "densed"))
    if c["set"] == "ragged":
        count = round(math.exp(rng.uniform(0, math.log(400))))
        c.update(count=count, elements=max(count, round(math.exp(rng.uniform(math.log(1000), math.log(2e8))))), sizes=rng.randrange(1 << 30))
    elif c["set"] == "stack":
        hidden = 64 * round(math.exp(rng.uniform(math.log(4), math.log(40))))
        c.update(hidden=hidden, layers=rng.randint(1, 4), vocab=round(math.exp(rng.uniform(math.log(100), math.log(32000)))))
    else:
        c.update(growth=rng.choice((8, 12, 16, 24, 32)), init=16 * rng.randint(1, 6))
    return c


def sizes_of(case):
    """the numbers of elements of the case's tensors, in order"""
    if case["set"] == "densed":             # DenseED with blocks [6, 8, 6]: normalisations in pairs and convolutions
        growth, c = case.get("growth", 16), case.get("init", 48)
        got = [c * 49]
        for block, layers in enumerate((6, 8, 6)):
            for _ in range(layers):
                got += [c, c, growth * c * 9]
                c += growth
            half = c // 2
            last = block == 2
            got += [c, c, half * c * (9 if last else 1), half, half]
            got += [half // 2 * half * 9, half // 2, half // 2, 3 * (half // 2) * 25] if last else [half * half * 9]
            c = half
        return got
    if case["set"] == "stack":              # an embedding, layers of four square products, a gated-free MLP, two norms; a norm
        d = case["hidden"]
        return [case["vocab"] * d] + [d * d, d * d, d * d, d * d, 4 * d * d, 4 * d * d, d, d] * case["layers"] + [d]
    r = random.Random(case["sizes"])
    w = [math.exp(r.uniform(0, 6)) for _ in range(case["count"])]
    got = [max(1, int(case["elements"] * x / sum(w))) for x in w]
    got[0] += max(0, case["elements"] - sum(got))
    return got


def work(case):
    n, item = sum(sizes_of(case)), DTYPES[case["dtype"]].itemsize
    if case["op"] == "clip":
        return {"bytes": n * item, "flops": 2 * n}
    weights = 2 * item + (4 if case["master"] else 0)
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (weights + item + states), "flops": 16 * n}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    sizes = sizes_of(case)
    dev = torch.device("cuda")
    gen = torch.Generator(dev)
    gen.manual_seed(seed)
    r = random.Random(seed)
    blocks = torch.tensor([-(-n // BLOCK) for n in sizes])
    first = torch.cumsum(blocks, 0) - blocks
    total = int(blocks.sum())
    tensor = torch.repeat_interleave(torch.arange(len(sizes)), blocks)            # of each block
    within = torch.arange(total) - first[tensor]
    filled = (torch.tensor(sizes)[tensor] - within * BLOCK).clamp(max=BLOCK)
    inside = (torch.arange(BLOCK, device=dev) < filled.to(dev)[:, None]).reshape(-1)
    size = total * BLOCK
    dtype = DTYPES[case["dtype"]]

    def normal():
        return torch.randn(size, generator=gen, device=dev)

    # gradients of very different sizes from tensor to tensor, a tenth of them zero (unused embeddings, cut activations)
    low, high = (-3.5, -2.0) if case["dtype"] == "float16" else (-5.0, -2.0)
    spread = torch.tensor([10.0 ** r.uniform(low, high) for _ in sizes])[tensor].to(dev).repeat_interleave(BLOCK) * inside
    g = (normal() * spread * (torch.rand(size, generator=gen, device=dev) > 0.1)).to(dtype)
    s = {"sizes": sizes, "g": g, "t": r.randint(50, 5000)}
    if case["op"] == "clip":
        s["limit"] = 2.0 * float(g.double().square().sum().sqrt())
        return s
    w = normal() * 0.03 * inside
    s["p"] = w.to(dtype)
    if case["master"]:
        bits = w.view(torch.int32)
        high16 = (bits + 0x8000) >> 16
        s["p"], s["low"] = high16.to(torch.int16).view(torch.bfloat16), (bits - (high16 << 16)).to(torch.int16)
    m = (0.4 * normal() + 0.1) * spread
    root = (torch.rand(size, generator=gen, device=dev) * 1.3 + 0.2) * spread
    if case["bits"] == 32:
        s["m"], s["v"] = m, root * root
    else:
        for x, q, scale in ((m, "mq", "ms"), (root, "rq", "rs")):
            rows = x.view(total, BLOCK)
            s[scale] = rows.abs().amax(1) * (1 / TOP)
            s[q] = (rows / s[scale].clamp(min=1e-30)[:, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(-1)
    s["tensor"], s["within"] = tensor.to(dev).int(), within.to(dev).int()
    s["limit"] = 0.7 * float(g.double().square().sum().sqrt()) if case["clip"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from pde_surrogate_amd import optim
        params, at, place = [], [], 0
        flat = s["p"] if "p" in s else torch.empty_like(s["g"])
        for n in s["sizes"]:
            at.append(slice(place, place + n))
            params.append(torch.nn.Parameter(flat[at[-1]]))
            params[-1].grad = s["g"][at[-1]]
            place += -(-n // BLOCK) * BLOCK
        s["params"] = params
        if case["op"] == "step":
            opt = optim.FusedAdamW(params, lr=LR, betas=(BETA1, case["beta2"]), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                   master_weights=case["master"], clip_norm=s["limit"], seed=SEED)
            saved = opt.state_dict()
            for i, a in enumerate(at):
                whole = slice(a.start, -(-a.stop // BLOCK) * BLOCK)
                rows = slice(a.start // BLOCK, whole.stop // BLOCK)
                st = {"step": torch.tensor(float(s["t"]))}
                if case["bits"] == 32:
                    st.update(exp_avg=s["m"][a], exp_avg_sq=s["v"][a])
                else:
                    st.update(exp_avg_q=s["mq"][whole], exp_avg_scale=s["ms"][rows], rms_q=s["rq"][whole], rms_scale=s["rs"][rows])
                if case["master"]:
                    st["low"] = s["low"][a]
                saved["state"][i] = st
            opt.load_state_dict(saved)
            s["opt"] = opt
            for k in ("m", "v", "mq", "ms", "rq", "rs", "low", "tensor", "within"):
                s.pop(k, None)
    return s


# ---- the operators -----------------------------------------------------------------------------------------------------
def run(s):
    if own:
        from pde_surrogate_amd import optim
        if s["case"]["op"] == "clip":
            return [optim.clip_grad_norm_(s["params"], s["limit"]), s["g"]]
        s["opt"].step()
        state = s["opt"].flat_state()
        names = ("exp_avg", "exp_avg_sq", "exp_avg_q", "exp_avg_scale", "rms_q", "rms_scale", "low")
        return [s["p"]] + [state[k][0] for k in names if k in state] + ([] if s["limit"] is None else [s["opt"].grad_norm])
    return plain_clip(s) if s["case"]["op"] == "clip" else plain_step(s)


def plain_clip(s):
    norm = s["g"].double().square().sum().sqrt().float()
    s["g"].copy_(s["g"].float() * (s["limit"] / (norm + 1e-6)).clamp(max=1.0))
    return [norm, s["g"]]


def mix(x):
    """of 32 bits held as int32: two multiplications between shifts"""
    a, b = MIX_A, MIX_B - (1 << 32)
    x = x ^ ((x >> 16) & 0xFFFF)
    x = x * a
    x = x ^ ((x >> 15) & 0x1FFFF)
    x = x * b
    return x ^ ((x >> 16) & 0xFFFF)


def dither(s):
    """20 bits for each element's m and 20 for its r"""
    gold = GOLD - (1 << 32)
    start = (SEED + GOLD * s["t"]) & 0xFFFFFFFF
    key = mix(torch.tensor(start - (1 << 32) if start >> 31 else start, dtype=torch.int32, device=s["g"].device))
    key = mix(key + (s["tensor"] + 1) * gold)
    key = mix(key + s["within"] * gold)
    h = mix(key[:, None] + torch.arange(BLOCK, dtype=torch.int32, device=key.device) * gold)
    return (h >> 12) & 0xFFFFF, h & 0xFFFFF


def held(x, noise):
    """(e4m3 codes of the non-negative rows x with their scales)"""
    top = x.amax(1, keepdim=True)
    live = top >= TINY
    inverse = torch.where(live, torch.full_like(top, TOP) / top, torch.zeros_like(top))
    y = x * inverse * 2.0 ** -120                  # e4m3's exponents now stand where float32's subnormal ones do
    code = ((y.view(torch.int32) + noise) >> 20).clamp(max=0x7E)
    return code, torch.where(live, top * (1 / TOP), torch.zeros_like(top)).view(-1)


def plain_step(s):
    c = s["case"]
    s["t"] += 1
    beta2, t = c["beta2"], s["t"]
    g, last = s["g"].float(), []
    if s["limit"] is not None:
        norm = s["g"].double().square().sum().sqrt().float()
        last = [norm]
        g = g * (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    if c["bits"] == 32:
        m = s["m"].mul_(BETA1).add_(g * (1 - BETA1))
        v = s["v"].mul_(beta2).add_(g * g * (1 - beta2))
        root, states = v.sqrt(), [m, v]
    else:
        g = g.view(-1, BLOCK)
        m = s["mq"].float().view(-1, BLOCK) * s["ms"][:, None] * BETA1 + g * (1 - BETA1)
        root = s["rq"].float().view(-1, BLOCK) * s["rs"][:, None]
        root = (root * root * beta2 + g * g * (1 - beta2)).sqrt()
        for_m, for_r = dither(s)
        code, s["ms"] = held(m.abs(), for_m)
        code = code | ((m.view(torch.int32) >> 24) & 0x80)
        s["mq"] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)
        code, s["rs"] = held(root, for_r)
        code = torch.maximum(code, (root > 0).int())            # a second moment that is not zero stays above zero
        s["rq"] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1)
        m, root, states = m.view(-1), root.view(-1), [s["mq"], s["ms"], s["rq"], s["rs"]]
    u = m / (root * (1 / math.sqrt(1 - beta2 ** t)) + EPS)
    if c["master"]:
        w = ((s["p"].view(torch.int16).int() << 16) + s["low"].int()).view(torch.float32)
    else:
        w = s["p"].float()
    w = w * (1 - LR * DECAY) - u * (LR / (1 - BETA1 ** t))
    if c["master"]:
        bits = w.view(torch.int32)
        high = (bits + 0x8000) >> 16
        s["p"].copy_(high.to(torch.int16).view(torch.bfloat16))
        s["low"].copy_((bits - (high << 16)).to(torch.int16))
        return [s["p"]] + states + [s["low"]] + last
    s["p"].copy_(w)
    return [s["p"]] + states + last


# ---- the same in 64 bits, from the formulas ----------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    g = s["g"].double()
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(g)
        return [norm, g * min(1.0, s["limit"] / (float(norm) + 1e-6))]
    t, last = s["t"] + 1, []
    if s["limit"] is not None:
        last = [torch.linalg.vector_norm(g)]
        g = g * min(1.0, s["limit"] / (float(last[0]) + 1e-6))
    w = s["p"].double()
    if case["master"]:
        # the low half counts steps of 2^-16 of the upper half's last place
        w = w + torch.ldexp(s["low"].double(), torch.frexp(s["p"].float().abs().clamp(min=2.0 ** -126))[1] - 24) * torch.where(torch.signbit(s["p"]), -1.0, 1.0)
    if case["bits"] == 32:
        m = BETA1 * s["m"].double() + (1 - BETA1) * g
        v = case["beta2"] * s["v"].double() + (1 - case["beta2"]) * g ** 2
        states = [m, v]
    else:
        m = BETA1 * (s["mq"].double().view(-1, BLOCK) * s["ms"].double()[:, None]).view(-1) + (1 - BETA1) * g
        v = case["beta2"] * (s["rq"].double().view(-1, BLOCK) * s["rs"].double()[:, None]).view(-1) ** 2 + (1 - case["beta2"]) * g ** 2
        states = _exact_states(s, t, m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK))
    hat = (v / (1 - case["beta2"] ** t)).sqrt() + EPS
    w = w - LR * DECAY * w - LR * (m / (1 - BETA1 ** t)) / hat
    return [w] + states + ([None] if case["master"] else []) + last


def _exact_states(s, t, m, root):
    full = (1 << 32) - 1

    def scramble(x):
        x = x ^ (x >> 16)
        x = (x * MIX_A) & full
        x = x ^ (x >> 15)
        x = (x * MIX_B) & full
        return x ^ (x >> 16)

    key = scramble((scramble((SEED + GOLD * t) & full) + GOLD * (s["tensor"].long() + 1)) & full)
    key = scramble((key + GOLD * s["within"].long()) & full)
    h = scramble((key[:, None] + GOLD * torch.arange(BLOCK, device=key.device)) & full)
    out = []
    for x, noise in ((m, h >> 12), (root, h & 0xFFFFF)):
        top = x.abs().amax(1, keepdim=True)
        scale = torch.where(top >= TINY, top / TOP, torch.zeros_like(top))
        y = torch.where(scale > 0, x.abs() / scale.clamp(min=1e-300), torch.zeros_like(x))
        place = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
        y = (torch.floor(y / place + noise.double() / (1 << 20)) * place).clamp(max=TOP)
        if x is root:
            y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
        out += [(torch.sign(x) * y).view(-1), scale.view(-1)]
    return out
