"""Cases, inputs, plain forms and exact values for three groups of operators of `ogmm_amd`:

  attention   cross attention to states of another length: ragged and masked keys, shared key / value heads, one query row or many, with gradients
  norm        root-mean-square norm with the residual's addition, its gradient, and its output in 8 bits (e4m3) with scales
  gradients   the global norm of many gradient tensors, and their clipping

`run` computes a case in plain torch operations in 32 bits, or, where `own` is true, by the framework's operators.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3_MAX = 448.0
NORM_EPS = 1e-6
CLIP_EPS = 1e-6


def listed():
    return [
        # one query token against one encoded cloud of 1024 points, four heads of 128 (the transformer's layout): all latency
        attention("attn one token", "fp16", B=1, Nq=1, Nk=1024, H=4, G=1, d=128),
        # single tokens of a batch of requests against long encoder states, eight query heads to a key head: the states' bytes
        attention("attn serving long states", "bf16", B=16, Nq=1, Nk=12288, H=32, G=8, d=128, lens=True),
        # a batch of registration pairs, 1024 points attending to the other cloud's 717, inference in 16 bits
        attention("attn pairs forward", "fp16", B=64, Nq=1024, Nk=717, H=4, G=1, d=128),
        # the same in the framework's own type, as a training step has it, clouds of different sizes padded to the largest
        attention("attn pairs training", "fp32", B=16, Nq=1024, Nk=717, H=4, G=1, d=128, lens=True, grad=True),
        # a decoder's training step against an encoder of another length, shared key heads, a mask over the encoder's positions
        attention("attn decoder training", "bf16", B=4, Nq=4096, Nk=2048, H=16, G=4, d=64, lens=True, mask=True, grad=True),
        # one token's row: all latency
        norm("norm one token", "bf16", R=1, D=512, residual=True),
        # a prompt's rows, quantised for storage: one scale a row
        norm("norm prompt 8 bits", "bf16", R=8192, D=4096, residual=True, q8=True),
        # an odd width, a scale to each 128 channels
        norm("norm odd groups 8 bits", "fp16", R=5000, D=717, residual=False, q8=True, group=128),
        # training on the feature maps of 128 clouds of 1024 points (64 pairs), forward and gradient
        norm("norm clouds training", "fp32", R=131072, D=512, residual=True, grad=True),
        # training in 16 bits with wide rows
        norm("norm wide training", "bf16", R=8192, D=8192, residual=True, grad=True),
        # the registration model's own gradients: 150 tensors of a hundred values to a million, 13 million in all; under the limit, as most steps are
        gradients("gradients of the model", "fp32", T=150, total=13_000_000, clip=False, out=False),
        # the gradients of a large model in 16 bits under a loss scale, clipped into the optimiser's 32-bit copies
        gradients("gradients large clipped", "bf16", T=400, total=300_000_000, clip=True, out=True),
    ]


def attention(name, dtype, B, Nq, Nk, H, G, d, lens=False, mask=False, grad=False):
    return {"name": name, "kind": "attention", "dtype": dtype, "B": B, "Nq": Nq, "Nk": Nk, "H": H, "G": G, "d": d, "lens": lens, "mask": mask, "grad": grad}


def norm(name, dtype, R, D, residual, q8=False, group=0, grad=False):
    return {"name": name, "kind": "norm", "dtype": dtype, "R": R, "D": D, "residual": residual, "q8": q8, "group": group, "grad": grad}


def gradients(name, dtype, T, total, clip, out):
    return {"name": name, "kind": "gradients", "dtype": dtype, "T": T, "total": total, "clip": clip, "out": out}


def log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "norm", "norm", "gradients"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "attention":
        while True:
            G, d = rng.choice([1, 1, 2, 4, 8]), rng.choice([32, 64, 64, 96, 128, 128])
            H = G * rng.choice([1, 2, 4, 8])
            few = rng.random() < 0.4
            Nq = rng.randint(1, 8) if few else log_between(rng, 9, 4096)
            Nk = log_between(rng, 1, 16384 if few else 4096)
            B = log_between(rng, 1, 64)
            grad = rng.random() < 0.5
            c = attention("", dtype, B, Nq, Nk, H, G, d, lens=rng.random() < 0.5, mask=rng.random() < 0.4, grad=grad)
            w = work(c)
            # (the plain form keeps several 32-bit maps of Nq x Nk scores)
            if w["flops"] <= 3.6e11 and w["bytes"] <= 8e8 and 4 * B * H * Nq * Nk <= 2.2e9:
                break
    elif kind == "norm":
        q8 = rng.random() < 0.4
        D = log_between(rng, 16, 12288)
        R = max(1, min(log_between(rng, 1, 200000), 67_000_000 // D))
        c = norm("", dtype, R, D, residual=rng.random() < 0.6, q8=q8, group=rng.choice([0, 0, 32, 64, 128]) if q8 else 0, grad=not q8 and rng.random() < 0.6)
    else:
        c = gradients("", dtype, log_between(rng, 1, 400), log_between(rng, 1000, 250_000_000), clip=rng.random() < 0.6, out=True)
        c["out"] = c["clip"] or rng.random() < 0.3
        c["total"] = max(c["total"], c["T"])
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": prepare_attention, "norm": prepare_norm, "gradients": prepare_gradients}[case["kind"]](case, g)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare_attention(case, g):
    B, Nq, Nk, H, G, d, dt = (case[k] for k in ("B", "Nq", "Nk", "H", "G", "d", "dtype"))
    dt = DTYPES[dt]
    s = {"case": case, "scale": d ** -0.5}
    s["q"] = (1.5 * randn(g, B, Nq, H, d)).to(dt)
    s["k"] = randn(g, B, Nk, H // G, d).to(dt)
    s["v"] = randn(g, B, Nk, H // G, d).to(dt)
    s["do"] = randn(g, B, Nq, H, d).to(dt) if case["grad"] else None
    # lengths between a half and the whole of the padded one; a mask that leaves seven of eight positions
    s["kv_lens"] = torch.randint((Nk + 1) // 2, Nk + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["lens"] else None
    s["key_mask"] = torch.rand(B, Nk, generator=g, device="cuda") < 0.875 if case["mask"] else None
    return s


def prepare_norm(case, g):
    R, D, dt = case["R"], case["D"], DTYPES[case["dtype"]]
    s = {"case": case}
    spread = torch.exp(0.5 * randn(g, R, 1))  # rows differ in size, as tokens do
    s["x"] = (randn(g, R, D) * spread).to(dt)
    s["r"] = (randn(g, R, D) * spread).to(dt) if case["residual"] else None
    s["w"] = (1.0 + 0.2 * randn(g, D)).to(dt)
    s["dy"] = randn(g, R, D).to(dt) if case["grad"] else None
    s["dh"] = randn(g, R, D).to(dt) if case["grad"] and case["residual"] else None
    return s


def tensor_sizes(T, total):
    """T sizes that add up to `total`, from single values to large matrices as the tensors of a model: a geometric row, every third a power of two, others odd"""
    weights = [math.exp(8.0 * ((37 * i) % T) / T) for i in range(T)]
    scale = (total - T) / sum(weights)
    sizes = [1 + int(w * scale) for w in weights]
    sizes = [1 << (n.bit_length() - 1) if i % 3 == 0 else n for i, n in enumerate(sizes)]
    sizes[-1] += total - sum(sizes)
    return sizes


def prepare_gradients(case, g):
    """The tensors are pieces of one bucket without gaps, as an all-reduce of gradients keeps them; so are the optimiser's 32-bit copies."""
    sizes = tensor_sizes(case["T"], case["total"])
    sizes_there = torch.tensor(sizes, device="cuda")
    levels = 10.0 ** -(torch.arange(case["T"], device="cuda") % 4).float()  # layers whose gradients differ in size by orders
    bucket = randn(g, case["total"]).mul_(torch.repeat_interleave(levels, sizes_there)).to(DTYPES[case["dtype"]])
    s = {"case": case, "bucket": bucket, "grads": list(bucket.split(sizes)), "inv_scale": 2.0 ** -6 if case["out"] else 1.0, "out": None}
    # the norm is below sqrt(total) times inv_scale: a limit well above it, or well below it
    s["max_norm"] = 2.0 * math.sqrt(case["total"]) if not case["clip"] else 1.0 if case["total"] >= 1_000_000 else 1e-4
    if case["out"]:
        s["bucket"] = torch.empty(case["total"], dtype=torch.float32, device="cuda")
        s["out"] = list(s["bucket"].split(sizes))
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": own_attention, "norm": own_norm, "gradients": own_gradients}[kind](state)
    return {"attention": plain_attention, "norm": plain_norm, "gradients": plain_gradients}[kind](state)


# ---------------------------------------------------------------------------------------------- the framework's operators
def own_attention(s):
    from ogmm_amd import ops, train_ops
    if not s["case"]["grad"]:
        return ops.cross_attention(s["q"], s["k"], s["v"], kv_lens=s["kv_lens"], key_mask=s["key_mask"], scale=s["scale"])
    q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
    o = train_ops.cross_attention(q, k, v, kv_lens=s["kv_lens"], key_mask=s["key_mask"], scale=s["scale"])
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def own_norm(s):
    from ogmm_amd import ops, train_ops
    case = s["case"]
    if case["q8"]:
        q, scales, h = ops.rms_norm_q8(s["x"], s["w"], residual=s["r"], eps=NORM_EPS, group=case["group"])
        return {"q": q, "scales": scales, "h": h if case["residual"] else None}
    if not case["grad"]:
        y, h, _ = ops.rms_norm(s["x"], s["w"], residual=s["r"], eps=NORM_EPS)
        return {"y": y, "h": h if case["residual"] else None}
    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    if not case["residual"]:
        y = train_ops.rms_norm(x, w, eps=NORM_EPS)
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    r = s["r"].detach().requires_grad_()
    y, h = train_ops.rms_norm(x, w, residual=r, eps=NORM_EPS)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dr": dr, "dw": dw}


def own_gradients(s):
    from ogmm_amd import ops
    total = ops.clip_grads_(s["grads"], s["max_norm"], inv_scale=s["inv_scale"], out=s["out"])
    return {"norm": total, "clipped": s["bucket"]}


# ---------------------------------------------------------------------------------------------- plain forms, in 32 bits
def admitted(s):
    """[B, Nk] truth values: the keys that a row may look at; None where that is all of them"""
    case = s["case"]
    ok = None
    if s["kv_lens"] is not None:
        ok = torch.arange(case["Nk"], device="cuda")[None, :] < s["kv_lens"][:, None]
    if s["key_mask"] is not None:
        ok = s["key_mask"] if ok is None else ok & s["key_mask"]
    return ok


def plain_attention(s):
    case = s["case"]
    B, Nq, Nk, H, G, d = (case[k] for k in ("B", "Nq", "Nk", "H", "G", "d"))
    Hkv = H // G
    ok = admitted(s)

    def heads_first(x, n):  # [B, n, Hkv * g, d] -> [B * Hkv, g * n, d]
        g = x.shape[2] // Hkv
        return x.float().view(B, n, Hkv, g, d).permute(0, 2, 3, 1, 4).reshape(B * Hkv, g * n, d)

    def points_first(x, n):
        g = x.shape[1] // n
        return x.view(B, Hkv, g, n, d).permute(0, 3, 1, 2, 4).reshape(B, n, Hkv * g, d).to(DTYPES[case["dtype"]])

    q, k, v = heads_first(s["q"], Nq) * s["scale"], heads_first(s["k"], Nk), heads_first(s["v"], Nk)
    scores = torch.bmm(q, k.transpose(1, 2))
    if ok is not None:
        ok = ok[:, None, None, :].expand(B, Hkv, 1, Nk).reshape(B * Hkv, 1, Nk)
        scores = scores.masked_fill(~ok, -math.inf)
    top = scores.amax(dim=2, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(dim=2, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = torch.bmm(p, v)
    if not case["grad"]:
        return points_first(o, Nq)
    do = heads_first(s["do"], Nq)
    dv = torch.bmm(p.transpose(1, 2), do)
    dp = torch.bmm(do, v.transpose(1, 2))
    ds = p * (dp - (do * o).sum(dim=2, keepdim=True))
    del p, dp
    dq = torch.bmm(ds, k) * s["scale"]
    dk = torch.bmm(ds.transpose(1, 2), q)
    return {"o": points_first(o, Nq), "dq": points_first(dq, Nq), "dk": points_first(dk, Nk), "dv": points_first(dv, Nk)}


def plain_norm(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    R, D = case["R"], case["D"]
    w = s["w"].float()
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + NORM_EPS)
    y = h * rstd * w
    stored = h.to(dt) if case["residual"] else None
    if case["q8"]:
        width = case["group"] or D
        pad = -D % width
        yg = torch.cat([y, y.new_zeros(R, pad)], dim=1).view(R, -1, width) if pad else y.view(R, -1, width)
        scales = yg.abs().amax(dim=2) / E4M3_MAX
        q = (yg / scales.masked_fill(scales == 0, 1.0)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
        return {"q": q.reshape(R, D + pad)[:, :D].to(torch.float8_e4m3fn), "scales": scales, "h": stored}
    if not case["grad"]:
        return {"y": y.to(dt), "h": stored}
    dy = s["dy"].float()
    xh = h * rstd
    g = dy * w
    dx = rstd * (g - xh * (g * xh).mean(dim=1, keepdim=True))
    dw = (dy.double() * xh.double()).sum(dim=0).to(dt)  # a sum over all rows
    if not case["residual"]:
        return {"y": y.to(dt), "dx": dx.to(dt), "dw": dw}
    dx = (dx + s["dh"].float()).to(dt)
    return {"y": y.to(dt), "h": stored, "dx": dx, "dr": dx, "dw": dw}


def plain_gradients(s):
    case = s["case"]
    squares = torch.stack([g.double().square().sum() for g in s["grads"]])  # sums over up to hundreds of millions of values
    total = (squares.sum().sqrt() * s["inv_scale"]).float()
    factor = (s["max_norm"] / (total + CLIP_EPS)).clamp(max=1.0) * s["inv_scale"]
    if case["out"]:
        for g, o in zip(s["grads"], s["out"]):
            torch.mul(g.float(), factor, out=o)
    else:
        for g in s["grads"]:
            g.mul_(factor)
    return {"norm": total, "clipped": s["bucket"]}


# ---------------------------------------------------------------------------------------------- what cannot be done without
def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "attention":
        B, Nq, Nk, H, G, d = (case[k] for k in ("B", "Nq", "Nk", "H", "G", "d"))
        part = (0.75 if case["lens"] else 1.0)  # mean share of the padded length; masked positions inside it are read and multiplied
        rows, states = B * Nq * H * d * e, part * B * Nk * (H // G) * d * e
        flops = 4.0 * part * B * H * Nq * Nk * d
        if not case["grad"]:
            return {"bytes": 2 * rows + 2 * states, "flops": flops}
        # forward and backward as one pass each: q, k, v twice, o and do; o, dq, dk, dv written
        return {"bytes": 2 * (rows + 2 * states) + 2 * rows + rows + rows + 2 * states, "flops": 3.5 * flops}
    if case["kind"] == "norm":
        R, D = case["R"], case["D"]
        n = R * D
        if case["q8"]:
            return {"bytes": n * (e + (2 * e if case["residual"] else 0) + 1) + 4 * R * (-(-D // (case["group"] or D))) + D * e, "flops": 6.0 * n}
        forward = n * e * (4 if case["residual"] else 2) + D * e
        if not case["grad"]:
            return {"bytes": forward, "flops": 5.0 * n}
        return {"bytes": forward + n * e * (4 if case["residual"] else 3) + 2 * D * e, "flops": 15.0 * n}
    n = case["total"]
    if case["out"]:
        return {"bytes": n * (2 * e + 4), "flops": 3.0 * n}  # the factor depends on every value: read, then read again and written
    return {"bytes": n * e, "flops": 2.0 * n}  # under the limit and unscaled: nothing changes


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": exact_attention, "norm": exact_norm, "gradients": exact_gradients}[case["kind"]](s)


def exact_attention(s):
    """The softmax over each row's admitted keys, one batch entry and key head at a time; gradients by torch's own differentiation."""
    case = s["case"]
    B, Nq, Nk, H, G, d = (case[k] for k in ("B", "Nq", "Nk", "H", "G", "d"))
    if B * H * Nq * Nk * (3 if case["grad"] else 1) > 4e9 or B * (H // G) > 600:
        return None
    names = ("o", "dq", "dk", "dv") if case["grad"] else ("o",)
    like = {"o": s["q"], "dq": s["q"], "dk": s["k"], "dv": s["v"]}
    out = {n: torch.zeros(like[n].shape, dtype=torch.float64, device="cuda") for n in names}
    lens = s["kv_lens"].tolist() if s["kv_lens"] is not None else [Nk] * B
    for b in range(B):
        keys = torch.arange(lens[b], device="cuda")
        if s["key_mask"] is not None:
            keys = keys[s["key_mask"][b, :lens[b]]]
        if not keys.numel():
            continue
        for j in range(H // G):
            mine = slice(j * G, (j + 1) * G)
            q = s["q"][b, :, mine].double().reshape(Nq * G, d)
            k, v = s["k"][b, keys, j].double(), s["v"][b, keys, j].double()
            if not case["grad"]:
                out["o"][b, :, mine] = (torch.softmax(q @ k.t() * s["scale"], dim=1) @ v).view(Nq, G, d)
                continue
            for t in (q, k, v):
                t.requires_grad_()
            o = torch.softmax(q @ k.t() * s["scale"], dim=1) @ v
            dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"][b, :, mine].double().reshape(Nq * G, d))
            out["o"][b, :, mine], out["dq"][b, :, mine] = o.detach().view(Nq, G, d), dq.view(Nq, G, d)
            out["dk"][b, keys, j], out["dv"][b, keys, j] = dk, dv
    return out if case["grad"] else out["o"]


def exact_norm(s):
    case, D = s["case"], s["case"]["D"]
    x, w = s["x"].double(), s["w"].double()
    h = x + s["r"].double() if case["residual"] else x
    if case["grad"]:
        h.requires_grad_()
        w.requires_grad_()
    y = w * h / ((h ** 2).sum(dim=1, keepdim=True) / D + NORM_EPS).sqrt()
    stored = h.detach() if case["residual"] else None
    if case["q8"]:
        width = case["group"] or D
        scales = torch.stack([y[:, i:i + width].abs().amax(dim=1) for i in range(0, D, width)], dim=1) / E4M3_MAX
        each = scales.repeat_interleave(width, dim=1)[:, :D]
        return {"q": nearest_e4m3(torch.where(each > 0, y / each, torch.zeros_like(y))), "scales": scales, "h": stored}
    if not case["grad"]:
        return {"y": y, "h": stored}
    dx, dw = torch.autograd.grad(y, (h, w), s["dy"].double())
    if not case["residual"]:
        return {"y": y.detach(), "dx": dx, "dw": dw}
    dx = dx + s["dh"].double()
    return {"y": y.detach(), "h": stored, "dx": dx, "dr": dx, "dw": dw}


def nearest_e4m3(x):
    """x rounded to the nearest value of four exponent and three mantissa bits (ties to even), in 64 bits"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact_gradients(s):
    case = s["case"]
    total = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in s["grads"])) * s["inv_scale"]
    factor = min(1.0, s["max_norm"] / (total + CLIP_EPS)) * s["inv_scale"]
    return {"norm": torch.tensor(total, dtype=torch.float64), "clipped": torch.cat([g.double() * factor for g in s["grads"]])}
