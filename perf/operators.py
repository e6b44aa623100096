"""Measured cases of the device-resident AdamW step (``GraphAdamW``) and of layer norm / RMS norm with their
backward passes, beside plain forms of the same operators in elementary torch operations.

``own`` selects which side ``run`` computes: the plain form, or the package's public calls.
"""

import math

import torch

own = False

BLOCK = 256           # values per scale of an 8-bit moment; every tensor starts on such a boundary in the flat buffers
SEED = 11             # of the stochastic rounding
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
STEPS_BEFORE = 100    # steps already taken: the state is one of mid-training
_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------- the cases

def listed():
    return [
        # One Llama-7B decoder layer (four 4096^2 projections, three MLP matrices, two norm weights), bf16 training:
        # what a step costs per layer with 8-bit and with fp32 moments.
        dict(name="adamw int8 decoder layer", op="adamw", state="int8", weights="bf16", clip=1, captured=0,
             sizes="16777216*4+45088768*3+4096*2"),
        dict(name="adamw fp32 decoder layer", op="adamw", state="fp32", weights="bf16", clip=1, captured=0,
             sizes="16777216*4+45088768*3+4096*2"),
        # The norm weights alone: the smallest step, where the calls' latency is all there is.
        dict(name="adamw int8 one norm weight", op="adamw", state="int8", weights="bf16", clip=0, captured=0,
             sizes="4096"),
        # A small fp32 model of many tensors of odd sizes (biases, norms, narrow matrices), its step captured into a
        # CUDA graph and replayed, as a program does whose steps are short.
        dict(name="adamw fp32 many odd tensors", op="adamw", state="fp32", weights="fp32", clip=1, captured=1,
             sizes="1*8+97*48+1023*48+4097*48+65537*24+300007*8"),
        # A mid-sized fp32 model whose tensors end inside blocks, vectors and tiles.
        dict(name="adamw int8 ragged fp32", op="adamw", state="int8", weights="fp32", clip=0, captured=0,
             sizes="5000011+1250001*6+130999*12+255*30+257*30"),
        # The norm of the training command's decoder: batch 8 x 512 tokens, hidden 4096, forward and backward.
        dict(name="rms norm train 4096x4096", op="rms", rows=4096, cols=4096, dtype="bf16", backward=1, pad=0),
        # Long batches of a wider model.
        dict(name="layer norm train 32768x8192", op="layer", rows=32768, cols=8192, dtype="bf16", backward=1, pad=0),
        # A single token of a forward pass.
        dict(name="layer norm one token", op="layer", rows=1, cols=4096, dtype="bf16", backward=0, pad=0),
        # A long prompt, forward only.
        dict(name="rms norm prompt 32768x4096", op="rms", rows=32768, cols=4096, dtype="bf16", backward=0, pad=0),
        # fp32 activations of an odd width, read out of a wider buffer (rows not contiguous).
        dict(name="layer norm train odd fp32", op="layer", rows=5003, cols=1023, dtype="fp32", backward=1, pad=5),
        # Narrow rows (per-head norms): many short reductions.
        dict(name="rms norm heads 262144x128", op="rms", rows=262144, cols=128, dtype="bf16", backward=1, pad=0),
        # Very wide rows, few of them.
        dict(name="layer norm train wide", op="layer", rows=515, cols=20000, dtype="bf16", backward=1, pad=0),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.45:
        parts, total = [], 0
        for _ in range(rng.randint(1, 6)):
            size, count = _between(rng, 1, 30_000_000), rng.randint(1, 40)
            count = max(1, min(count, 100_000_000 // size))
            if total + size * count > 150_000_000:
                continue
            total += size * count
            parts.append("%d*%d" % (size, count))
        return dict(op="adamw", state=rng.choice(("int8", "fp32")), weights=rng.choice(("bf16", "fp32")),
                    clip=rng.randint(0, 1), captured=rng.choice((0, 0, 0, 1)), sizes="+".join(parts) or "4097")
    cols = _between(rng, 16, 24_000)
    if rng.random() < 0.5:
        cols = -(-cols // 8) * 8
    rows = min(_between(rng, 1, 300_000), max(1, 120_000_000 // cols))
    return dict(op=rng.choice(("layer", "rms")), rows=rows, cols=cols, dtype=rng.choice(("bf16", "bf16", "fp32")),
                backward=rng.randint(0, 1), pad=rng.choice((0, 0, 8, 3)))


def _sizes(case):
    out = []
    for part in case["sizes"].split("+"):
        size, _, count = part.partition("*")
        out += [int(size)] * int(count or 1)
    return out


def _starts(sizes):
    """Where each tensor starts in the flat buffers, and their length: whole blocks per tensor."""
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


# --------------------------------------------------------------------------- inputs

def _adamw_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    sizes = _sizes(case)
    starts, total = _starts(sizes)
    dt = _DTYPE[case["weights"]]
    s = dict(case=case, sizes=sizes, starts=starts, total=total, step=STEPS_BEFORE)
    # which elements belong to a tensor: the rest of each last block is padding, zero throughout
    n = torch.tensor(sizes, device=dev)
    blocks = (n + BLOCK - 1) // BLOCK
    owner = torch.repeat_interleave(torch.arange(len(sizes), device=dev), blocks)     # tensor of each block
    first = torch.tensor(starts, device=dev)[owner]
    left = (n[owner] - (torch.arange(total // BLOCK, device=dev) * BLOCK - first)).clamp(max=BLOCK)
    s["owner"], s["start_of_block"] = owner, first

    def zero_padding(flat):
        rows = flat.view(-1, BLOCK)
        short = torch.nonzero(left < BLOCK).squeeze(1)
        rows[short] = torch.where(torch.arange(BLOCK, device=dev) < left[short, None], rows[short],
                                  torch.zeros((), dtype=flat.dtype, device=dev))
        return flat

    master = zero_padding(torch.empty(total, device=dev).normal_(0.0, 0.02, generator=gen))
    s["grad"] = zero_padding(torch.empty(total, dtype=dt, device=dev).normal_(0.0, 1e-3, generator=gen))
    if dt == torch.bfloat16:
        s["master"], s["weight"] = master, master.to(dt)
    else:
        s["master"], s["weight"] = None, master
    scale = lambda low, high: torch.empty(total // BLOCK, device=dev).uniform_(low, high, generator=gen)   # noqa: E731
    if case["state"] == "int8":
        s["m"] = zero_padding(torch.randint(-127, 128, (total,), dtype=torch.int8, device=dev, generator=gen))
        s["v"] = zero_padding(torch.randint(1, 256, (total,), dtype=torch.uint8, device=dev, generator=gen))
        s["m_scale"], s["v_scale"] = scale(2e-6, 8e-6), scale(3e-6, 1.2e-5)
    else:
        s["m"] = zero_padding(torch.empty(total, device=dev).normal_(0.0, 3e-4, generator=gen))
        s["v"] = zero_padding(torch.empty(total, device=dev).uniform_(1e-8, 4e-6, generator=gen))
    s["scale"] = torch.empty(1, device=dev).uniform_(0.3, 0.9, generator=gen) if case["clip"] else None
    return s


def _norm_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, cols, dt = case["rows"], case["cols"], _DTYPE[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(mean, std, generator=gen)

    # activations: channels of their own offset, one in about a hundred of them large
    x = normal(rows, cols + case["pad"])
    loud = torch.rand(cols + case["pad"], device=dev, generator=gen) < 0.01
    x.mul_(torch.where(loud, 20.0, 1.0).to(dt)).add_(normal(cols + case["pad"], std=0.3))
    s = dict(case=case, x=x[:, :cols], w=normal(cols, std=0.1, mean=1.0))
    if case["op"] == "layer":
        s["b"] = normal(cols, std=0.1)
    if case["backward"]:
        s["dy"] = normal(rows, cols, std=1e-2)
    return s


def prepare(case, seed):
    if case["op"] != "adamw":
        s = _norm_inputs(case, seed)
        if case["backward"]:
            for name in ("x", "w", "b"):
                if name in s:
                    s[name].requires_grad_(True)
        return s
    s = _adamw_inputs(case, seed)
    if own:   # the program's optimizer, at the same point of its training
        import adambridge_b200 as ab
        params = []
        for at, n in zip(s["starts"], s["sizes"]):
            p = torch.nn.Parameter(s["weight"][at:at + n])
            p.grad = s["grad"][at:at + n]
            params.append(p)
        s["opt"] = opt = ab.GraphAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                                       precision=case["state"], stochastic_rounding=True, seed=SEED)
        opt.prepare()
        arena = opt.arenas[0]
        for name in ("master", "m", "v", "m_scale", "v_scale"):
            if s.get(name) is not None:
                getattr(arena, name).copy_(s[name])
        arena.steps.fill_(STEPS_BEFORE)
        if case["captured"]:
            s["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(s["graph"]):
                opt.step(grad_scale=s["scale"])
    return s


# --------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if own:
        import adambridge_b200 as ab
        if case["op"] == "adamw":
            if case["captured"]:
                s["graph"].replay()
            else:
                s["opt"].step(grad_scale=s["scale"])
            arena = s["opt"].arenas[0]
            return _adamw_outputs(s["weight"], arena.master, arena.exp_avg(), arena.exp_avg_sq())
        if not case["backward"]:
            with torch.no_grad():
                if case["op"] == "rms":
                    return {"y": ab.rms_norm(s["x"], s["w"], eps=1e-5)}
                return {"y": ab.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)}
        if case["op"] == "rms":
            y = ab.rms_norm(s["x"], s["w"], eps=1e-5)
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        y = ab.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["op"] == "adamw":
        return _adamw_plain(s)
    with torch.no_grad():
        return _norm_plain(s)


def _adamw_outputs(weight, master, m, v):
    out = {"weight": weight, "exp_avg": m, "exp_avg_sq": v}
    if master is not None:
        out["master"] = master
    return out


def _hash(x):
    """A 32-bit integer hash (two multiply-xorshift rounds) of whole numbers below 2^32, held in 64 bits."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_words(s):
    """The rounding's 32 random bits of every element: a hash of its place in its tensor, the tensor and the step."""
    stream = _hash(_hash(_hash(torch.full_like(s["owner"], SEED)) ^ s["owner"]) ^ s["step"])        # per block
    place = torch.arange(s["total"], device=s["grad"].device).view(-1, BLOCK) - s["start_of_block"][:, None]
    return _hash((place & 0xFFFFFFFF) ^ stream[:, None])


def _decoded(s):
    if s["case"]["state"] == "fp32":
        return s["m"], s["v"]
    m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
    r = s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]
    return m, (r * r).view(-1)


def _adamw_plain(s):
    """The step in elementary operations, every one rounded to 32 bits; the state is updated in place."""
    s["step"] += 1
    t = s["step"]
    step_size, root = LR / (1 - BETAS[0] ** t), 1 / math.sqrt(1 - BETAS[1] ** t)
    m, v = _decoded(s)
    g = s["grad"].float()
    if s["scale"] is not None:
        g = g * s["scale"]
    p = s["weight"] if s["master"] is None else s["master"]
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + g * (1 - BETAS[1]) * g
    r = torch.sqrt(v)
    p.copy_(p * (1 - LR * DECAY) - m / (r * root + EPS) * step_size)
    if s["master"] is not None:
        s["weight"].copy_(p)
    if s["case"]["state"] == "fp32":
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        words = _random_words(s)
        um, uv = (words & 0xFFFF).float() / 65536, (words >> 16).float() / 65536
        del words
        m, r = m.view(-1, BLOCK), r.view(-1, BLOCK)
        # just below 127 and 255, so that no product of a value with its block's factor rounds above them
        top_m, top_r = m.abs().amax(1), r.amax(1)
        bound = torch.tensor([127.0, 255.0], device=m.device).nextafter(torch.zeros(2, device=m.device))
        to_m = torch.where(top_m > 2.0 ** -100, bound[0] / top_m, 0.0)
        to_r = torch.where(top_r > 2.0 ** -100, bound[1] / top_r, 0.0)
        s["m"].copy_(torch.floor(m * to_m[:, None] + um).view(-1))
        x = r * to_r[:, None]
        q = torch.floor(x)
        q = q + ((x - q) * (x + q) > uv * (q + q + 1)).float()
        s["v"].copy_(torch.where(r > 0, torch.clamp(q, min=1), q).view(-1))
        s["m_scale"].copy_(torch.where(top_m > 2.0 ** -100, top_m * (1 / 127), 0.0))
        s["v_scale"].copy_(torch.where(top_r > 2.0 ** -100, top_r * (1 / 255), 0.0))
    m, v = _decoded(s)
    return _adamw_outputs(s["weight"], s["master"], m, v)


def _norm_plain(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    if case["op"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    h = x * r
    y = h * w
    if case["op"] == "layer":
        y = y + s["b"].float()
    out = {"y": y.to(s["x"].dtype)}
    if case["backward"]:
        dy = s["dy"].float()
        a = dy * w
        dx = a - h * (a * h).mean(-1, keepdim=True)
        if case["op"] == "layer":
            dx = dx - a.mean(-1, keepdim=True)
            out["db"] = dy.sum(0).to(s["b"].dtype)
        out["dx"] = (dx * r).to(s["x"].dtype)
        out["dw"] = (dy * h).sum(0).to(s["w"].dtype)
    return out


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        wide = case["weights"] == "bf16"
        per = (2 + 2 + 8) if wide else (4 + 8)            # gradient in, weight out, parameter in and out
        # 8-bit: codes in and out, and the values that they stand for out, as fp32; else the moments in and out
        per += (4 + 16 / BLOCK + 8) if case["state"] == "int8" else 16
        return {"bytes": n * per, "flops": n * 20}
    n, size = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
    params = case["cols"] * size * (2 if case["op"] == "layer" else 1)
    if case["backward"]:   # x and dy in, y and dx out
        return {"bytes": n * size * 4 + 2 * params, "flops": n * 20}
    return {"bytes": n * size * 2 + params, "flops": n * 8}


# --------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    if case["op"] == "adamw":
        s = _adamw_inputs(case, seed)
        t = STEPS_BEFORE + 1
        b1, b2 = BETAS
        if case["state"] == "int8":
            block = torch.arange(s["total"], device="cuda") // BLOCK
            m = s["m"].double() * s["m_scale"].double()[block]
            v = (s["v"].double() * s["v_scale"].double()[block]).square()
            del block
        else:
            m, v = s["m"].double(), s["v"].double()
        g = s["grad"].double()
        if s["scale"] is not None:
            g = g * s["scale"].double()
        p = (s["weight"] if s["master"] is None else s["master"]).double()
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).addcmul_(g, g, value=1 - b2)
        p.mul_(1 - LR * DECAY).addcdiv_(m / (1 - b1 ** t), (v / (1 - b2 ** t)).sqrt().add_(EPS), value=-LR)
        # an 8-bit moment is one of two neighbouring codes, by its random bits: there is no 64-bit value of it
        kept = case["state"] == "fp32"
        return _adamw_outputs(p, None if s["master"] is None else p, m if kept else None, v if kept else None)
    s = _norm_inputs(case, seed)
    x, w = s["x"].detach().double(), s["w"].double()
    mu = x.mean(1) if case["op"] == "layer" else torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    dev = ((x - mu[:, None]).square().sum(1) / case["cols"] + 1e-5).sqrt()
    hat = (x - mu[:, None]) / dev[:, None]
    del x
    out = {"y": hat * w + (s["b"].double() if case["op"] == "layer" else 0.0)}
    if case["backward"]:
        dy = s["dy"].double()
        out["dw"] = torch.einsum("rc,rc->c", dy, hat)
        a = dy * w
        mean_a = a.mean(1, keepdim=True) if case["op"] == "layer" else 0.0
        out["dx"] = (a - mean_a - hat * ((a * hat).sum(1, keepdim=True) / case["cols"])) / dev[:, None]
        if case["op"] == "layer":
            out["db"] = dy.sum(0)
    return out
