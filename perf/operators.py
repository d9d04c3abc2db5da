"""Cases and plain forms of the sequence and clipping operators: rotary positions with several axes
(`embedding.rotary`), attention with capped scores, distance bias and interval masks
(`attention.span_attention`), the global gradient norm with clipping, alone (`optim.clip_grad_norm_`) and
inside the Adam step (`optim.adam_step_`).

`run(state)` computes one pass, in elementary torch operations or, where `own` is true, through the package.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------

def _attend(name, kind, batch, nq, nk, heads, kv, dim, mask, cap=0.0, slopes=False, train=True):
    return {"name": name, "op": "attend", "type": kind, "batch": batch, "nq": nq, "nk": nk, "heads": heads, "kv": kv, "dim": dim,
            "mask": mask, "cap": cap, "slopes": slopes, "train": train}


def _rotate(name, kind, batch, axes, sizes, heads, kv, dim, interleaved=False, train=False, offset=0):
    return {"name": name, "op": "rotate", "type": kind, "batch": batch, "axes": axes, "sizes": sizes, "heads": heads, "kv": kv,
            "dim": dim, "interleaved": interleaved, "train": train, "offset": offset}


def listed():
    return [
        # attention over the 7x7 feature map at the bottom of a 28x28 network, one image: launch latency
        _attend("attend 7x7 map, one image", "fp32", 1, 49, 49, 4, 4, 32, "none"),
        # a training batch over 32x32 pixels in the network's own type, scores capped
        _attend("attend 32x32 pixels, training", "fp32", 32, 1024, 1024, 4, 4, 32, "none", cap=30.0),
        # label or text tokens in front of 45x45 pixels: the prefix sees itself, the pixels follow one by one; odd length
        _attend("attend prefix and pixels", "bf16", 4, 2125, 2125, 16, 16, 64, "prefix", cap=50.0),
        # images of different sizes packed into one sequence, shared key/value heads, distance bias
        _attend("attend packed images", "bf16", 1, 8192, 8192, 16, 4, 128, "documents", slopes=True),
        # a 128x128 image at once, inference
        _attend("attend 128x128 pixels", "bf16", 1, 16384, 16384, 8, 8, 128, "none", train=False),
        # single tokens of a ragged batch against their key/value buffers
        _attend("attend one token, batch", "bf16", 32, 1, 8192, 32, 8, 128, "lengths", slopes=True, train=False),
        # two single tokens against long buffers, an odd head size: few rows, a long axis
        _attend("attend one token, long", "fp16", 2, 1, 65536, 16, 2, 80, "lengths", cap=50.0, train=False),
        # positions of one new token of each sequence of a batch, far along: launch latency
        _rotate("rotate one token", "bf16", 16, "32,48,48", "1,1,1", 32, 8, 128, offset=100000),
        # positions of 16 frames of 64x64 with their gradient, shared key heads
        _rotate("rotate 16 frames, training", "bf16", 1, "32,48,48", "16,64,64", 16, 4, 128, train=True),
        # the clipped optimizer step of the smallest network of the tests: many tiny tensors
        {"name": "clipped step, tiny network", "op": "step", "unet": 8, "emb": 16, "max_norm": 1.0},
        # the clipped optimizer step of the full second-iteration network
        {"name": "clipped step, full network", "op": "step", "unet": 64, "emb": 128, "max_norm": 1.0},
        # clipping alone over a large list of tensors of two types, ragged sizes
        {"name": "clip 400 tensors, two types", "op": "clip", "tensors": 400, "largest": 1 << 21, "type": "mixed", "max_norm": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "token", "rotate", "rotate", "step", "clip"])
    kind = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "attend":
        while True:
            mask = rng.choice(["none", "causal", "prefix", "documents", "lengths"])
            n, batch = _log(rng, 1, 8192), _log(rng, 1, 32)
            if mask == "documents":
                batch = 1
            kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
            dim = 8 * rng.randint(2, 16)
            c = _attend("", kind, batch, n, n, kv * group, kv, dim, mask, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                        slopes=rng.random() < 0.4, train=rng.random() < 0.6)
            pairs = batch * kv * group * n * n
            # the plain form holds several arrays of this many values
            if pairs <= (1 << 27 if kind == "fp32" else 1 << 30) and pairs * dim * 14 <= 1e12:
                break
    elif op == "token":
        while True:
            batch, nk = _log(rng, 1, 64), _log(rng, 1, 65536)
            kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 5, 8])
            dim = 8 * rng.randint(2, 16)
            nq = rng.choice([1, 1, 1, 2, 5])
            if nk >= nq and batch * kv * nk * dim <= 1 << 27 and batch * kv * group * nk * dim <= 1 << 30:
                break
        c = _attend("", kind, batch, nq, nk, kv * group, kv, dim, "lengths", cap=rng.choice([0.0, 50.0]), slopes=rng.random() < 0.5, train=False)
    elif op == "rotate":
        while True:
            count = rng.randint(1, 3)
            axes = [2 * rng.randint(1, 32) for _ in range(count)]
            dim = 8 * ((sum(axes) + 7) // 8) + 8 * rng.randint(0, 2)
            sizes = [_log(rng, 1, 64) for _ in range(count)]
            heads = rng.choice([1, 2, 4, 8, 16, 24])
            batch = _log(rng, 1, 16)
            if dim <= 128 and batch * math.prod(sizes) * heads * dim <= 1 << 25:
                break
        c = _rotate("", kind, batch, ",".join(map(str, axes)), ",".join(map(str, sizes)), heads, rng.choice([h for h in (1, 2, 4, heads) if heads % h == 0]),
                    dim, interleaved=rng.random() < 0.5, train=rng.random() < 0.5, offset=rng.choice([0, 0, 1000, 200000]))
    elif op == "step":
        c = {"op": "step", "unet": 8 * _log(rng, 1, 12), "emb": 4 * rng.randint(4, 64), "max_norm": rng.choice([0.5, 1.0, 5.0, 1e4])}
    else:
        c = {"op": "clip", "tensors": _log(rng, 1, 500), "largest": _log(rng, 1, 1 << 20), "type": rng.choice(["fp32", "bf16", "fp16", "mixed"]),
             "max_norm": rng.choice([0.5, 1.0, 5.0, 1e6])}
    c.pop("name", None)
    return c


# ---- sizes that follow from a case ---------------------------------------------------------------------------------

def _spans(c):
    """The keys [first, last) that each row sees: int32 [batch][nq][2], or None; and each row's position, or None. The same
    for every seed, so that `work` can count the pairs."""
    batch, nq, nk = c["batch"], c["nq"], c["nk"]
    r = np.random.RandomState(nq + 31 * nk + 977 * batch)
    i = np.arange(nq)
    if c["mask"] == "prefix":
        p = r.randint(0, max(1, nk // 8) + 1, (batch, 1))
        hi = np.minimum(np.maximum(i[None] + 1, p), nk)
        return np.stack([np.zeros_like(hi), hi], -1).astype(np.int32), None
    if c["mask"] == "documents":
        cuts = np.unique(r.randint(0, nk + 1, max(1, nk // 340)))
        cuts = np.unique(np.concatenate([[0], cuts, [nk]]))
        d = np.searchsorted(cuts, i, side="right") - 1
        return np.broadcast_to(np.stack([cuts[d], cuts[d + 1]], -1), (batch, nq, 2)).astype(np.int32).copy(), None
    if c["mask"] == "lengths":
        length = r.randint(nk // 2, nk + 1, (batch, 1))
        length[0] = nk
        if batch > 2:
            length[-1] = min(1, nk)
        if nq == nk:                                             # a padded batch: rows past the end see nothing
            hi = np.where(i[None] < length, length, 0)
            return np.stack([np.zeros_like(hi), hi], -1).astype(np.int32), None
        pos = length - nq + i[None]                              # the last nq tokens of each sequence
        hi = np.clip(pos + 1, 0, nk)
        return np.stack([np.zeros_like(hi), hi], -1).astype(np.int32), pos.astype(np.int32)
    return None, None


def _pairs(c):
    """Visible (row, key) pairs of one head, and the keys that any row sees, over the batch."""
    if c["mask"] == "none":
        return c["batch"] * c["nq"] * c["nk"], c["batch"] * c["nk"]
    if c["mask"] == "causal":
        return c["batch"] * c["nq"] * (c["nq"] + 1) // 2, c["batch"] * c["nk"]
    s = _spans(c)[0].astype(np.int64)
    return int(np.maximum(s[..., 1] - s[..., 0], 0).sum()), int(s[..., 1].max(axis=1).sum())


def _unet(base, emb):
    """Element counts of the parameters of the second-iteration network, in its order."""
    n = []
    for m in (1, 2, 4, 8):
        n += [base * m * emb, base * m]

    def double(ci, co):
        for a, b in ((ci, co), (co, co), (co, co)):
            n.extend([a * b * 9, b, b, b])                       # convolution, its bias, the norm's scale and shift

    def attention(ch):
        n.extend([1, ch // 8 * ch, ch // 8, ch // 8 * ch, ch // 8, ch * ch, ch])

    double(1, base)
    for m in (1, 2):
        double(base * m, 2 * base * m)
        attention(2 * base * m)
    double(4 * base, 8 * base)
    attention(8 * base)
    for m in (8, 4, 2):
        n.extend([base * m * (base * m // 2) * 4, base * m // 2])
        double(base * m, base * m // 2)
        attention(base * m // 2)
    return n + [base, 1]


def _tensors(c):
    """(element count, type) of each tensor of a clipping case."""
    if c["op"] == "step":
        return [(n, "fp32") for n in _unet(c["unet"], c["emb"])]
    r = random.Random(c["tensors"] * 131 + c["largest"])
    kinds = ("fp32", "bf16") if c["type"] == "mixed" else (c["type"],)
    return [(_log(r, 1, c["largest"]) if i else c["largest"], kinds[i % len(kinds)]) for i in range(c["tensors"])]


def work(case):
    c = case
    if c["op"] == "attend":
        pairs, keys = _pairs(c)
        e, rows = BYTES[c["type"]], c["batch"] * c["nq"] * c["heads"] * c["dim"]
        kv = 2 * keys * c["kv"] * c["dim"]
        # forward: q, k, v read, out written; with the gradient: dout read, and dq, dk, dv written
        return {"bytes": e * (2 * rows + kv + ((2 * rows + kv) if c["train"] else 0)),
                "flops": pairs * c["heads"] * c["dim"] * (14 if c["train"] else 4)}
    if c["op"] == "rotate":
        tokens = c["batch"] * math.prod(map(int, c["sizes"].split(",")))
        n = tokens * (c["heads"] + c["kv"]) * c["dim"] * (2 if c["train"] else 1)
        return {"bytes": 2 * n * BYTES[c["type"]], "flops": 3 * n}
    sizes = _tensors(c)
    total = sum(n for n, _ in sizes)
    if c["op"] == "step":
        return {"bytes": 28 * total, "flops": 16 * total}          # g, p, m, v read; p, m, v written
    return {"bytes": sum(2 * n * BYTES[k] for n, k in sizes), "flops": 3 * total}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, kind=None):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[kind or c["type"]])

    s = {"case": c}
    if c["op"] == "attend":
        s["q"] = normal(c["batch"], c["nq"], c["heads"], c["dim"], scale=1.5)
        s["k"] = normal(c["batch"], c["nk"], c["kv"], c["dim"], scale=1.5)
        s["v"] = normal(c["batch"], c["nk"], c["kv"], c["dim"])
        if c["train"]:
            s["dout"] = normal(c["batch"], c["nq"], c["heads"], c["dim"])
            for name in ("q", "k", "v"):
                s[name].requires_grad_(True)
        spans, positions = _spans(c)
        s["spans"] = None if spans is None else torch.from_numpy(spans).cuda()
        s["positions"] = None if positions is None else torch.from_numpy(positions).cuda()
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, c["heads"] + 1, dtype=torch.float64) / c["heads"])).float().cuda() if c["slopes"] else None
    elif c["op"] == "rotate":
        sizes = [int(n) for n in c["sizes"].split(",")]
        grid = torch.cartesian_prod(*[torch.arange(n) for n in sizes]).reshape(-1, len(sizes)) + c["offset"]
        # a batch of separate sequences stands at positions of its own
        shift = torch.randint(0, 64, (c["batch"], 1, len(sizes)), generator=torch.Generator().manual_seed(seed))
        s["positions"] = (grid[None] + shift).to(torch.int32).cuda()
        s["axes"] = tuple(int(n) for n in c["axes"].split(","))
        n = grid.shape[0]
        s["q"] = normal(c["batch"], n, c["heads"], c["dim"])
        s["k"] = normal(c["batch"], n, c["kv"], c["dim"])
        if c["train"]:
            s["dq"] = normal(c["batch"], n, c["heads"], c["dim"])
            s["dk"] = normal(c["batch"], n, c["kv"], c["dim"])
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
    else:
        # gradients as a data-parallel step leaves them: slices of one flat buffer for each type, each on a 256-byte boundary
        sizes = _tensors(c)
        s["flat"], at = {}, {}
        for kind in sorted({k for _, k in sizes}):
            room = sum(-(-n // 128) * 128 for n, k in sizes if k == kind)
            s["flat"][kind] = normal(room, scale=0.05, kind=kind)
            at[kind] = 0
        s["grads"], s["params"] = [], []
        flat = {"p": torch.zeros_like(s["flat"]["fp32"]), "m": torch.zeros_like(s["flat"]["fp32"]), "v": torch.zeros_like(s["flat"]["fp32"])} if c["op"] == "step" else {}
        if flat:
            room = flat["p"].numel()
            flat["p"].copy_(normal(room, scale=0.05, kind="fp32"))
            flat["m"].copy_(normal(room, scale=0.01, kind="fp32"))
            flat["v"].copy_(normal(room, scale=0.01, kind="fp32").square())
            s.update(flat_p=flat["p"], flat_m=flat["m"], flat_v=flat["v"], m=[], v=[], step=10)
        keep = {kind: torch.zeros(f.numel(), dtype=torch.bool) for kind, f in s["flat"].items()}
        for n, kind in sizes:
            o = at[kind]
            at[kind] += -(-n // 128) * 128
            keep[kind][o:o + n] = True
            s["grads"].append(s["flat"][kind][o:o + n])
            if flat:
                s["params"].append(flat["p"][o:o + n])
                s["m"].append(flat["m"][o:o + n])
                s["v"].append(flat["v"][o:o + n])
            else:
                p = torch.nn.Parameter(torch.empty(n, dtype=TYPES[kind], device="cuda"))
                p.grad = s["grads"][-1]
                s["params"].append(p)
        for kind, f in s["flat"].items():                         # the gaps between the slices hold zeros
            f.mul_(keep[kind].cuda())
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _plain_attend(s):
    c = s["case"]
    group = c["heads"] // c["kv"]
    scale = c["dim"] ** -0.5
    q = s["q"].detach().float().transpose(1, 2).contiguous()                                         # [B][H][nq][D]
    k = s["k"].detach().float().transpose(1, 2).repeat_interleave(group, 1).contiguous()
    v = s["v"].detach().float().transpose(1, 2).repeat_interleave(group, 1).contiguous()
    t = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    th = None
    if c["cap"]:
        th = torch.tanh(t.div_(c["cap"]))
        t = th * c["cap"]
    j = torch.arange(c["nk"], device=q.device)
    i = s["positions"].long() if s["positions"] is not None else (torch.arange(c["nq"], device=q.device) + c["nk"] - c["nq"])[None]
    if s["slopes"] is not None:
        t -= s["slopes"][None, :, None, None] * (i[:, None, :, None] - j).abs()
    if s["spans"] is not None:
        seen = (j >= s["spans"][:, None, :, :1]) & (j < s["spans"][:, None, :, 1:])
        t.masked_fill_(~seen, -math.inf)
    if c["mask"] == "causal":
        t.masked_fill_(j > i[:, None, :, None], -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp_(t.sub_(torch.where(torch.isinf(top), 0.0, top)))
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(s["q"].dtype).contiguous()
    if not c["train"]:
        return [out]
    do = s["dout"].float().transpose(1, 2).contiguous()

    def shared(x):                                                # the gradient of a shared head is the sum over its users
        return x.reshape(c["batch"], c["kv"], group, c["nk"], c["dim"]).sum(2).transpose(1, 2).to(s["k"].dtype).contiguous()

    dv = shared(torch.matmul(p.transpose(2, 3).contiguous(), do))
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if th is not None:
        ds.mul_(1 - th * th)
    ds.mul_(scale)
    dq = torch.matmul(ds, k).transpose(1, 2).to(s["q"].dtype).contiguous()
    dk = shared(torch.matmul(ds.transpose(2, 3).contiguous(), q))
    return [out, dq, dk, dv]


def _plain_rotate(s):
    c = s["case"]
    dev = s["q"].device
    half = [d // 2 for d in s["axes"]]
    freq = torch.cat([10000.0 ** (-2.0 * torch.arange(h, dtype=torch.float64, device=dev) / (2 * h)) for h in half])
    axis = torch.cat([torch.full((h,), a, dtype=torch.long, device=dev) for a, h in enumerate(half)])
    start = torch.cat([torch.full((h,), sum(s["axes"][:a]), dtype=torch.long, device=dev) for a, h in enumerate(half)])
    at = torch.cat([torch.arange(h, device=dev) for h in half])
    width = torch.cat([torch.full((h,), h, dtype=torch.long, device=dev) for h in half])
    one = start + (2 * at if c["interleaved"] else at)            # the two channels of each pair
    two = one + (1 if c["interleaved"] else width)
    angle = s["positions"].double()[..., axis] * freq             # [B][N][pairs], 64 bits: far positions turn many times
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def turn(x, sin):
        f = x.detach().float()
        y = f.clone()
        y[..., one] = f[..., one] * cos - f[..., two] * sin
        y[..., two] = f[..., two] * cos + f[..., one] * sin
        return y.to(x.dtype)

    out = [turn(s["q"], sin), turn(s["k"], sin)]
    return out + [turn(s["dq"], -sin), turn(s["dk"], -sin)] if c["train"] else out


def _plain_clip(s):
    c = s["case"]
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    coef = torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0)
    if c["op"] == "clip":
        done = [g.copy_(g.float() * coef) for g in s["grads"]]
        return {"norm": norm, **s["flat"]}
    s["step"] += 1
    lr, b1, b2, eps = 2e-4, 0.9, 0.999, 1e-8
    size, root = lr / (1 - b1 ** s["step"]), math.sqrt(1 - b2 ** s["step"])
    grads = [g * coef for g in s["grads"]]
    done = [m.mul_(b1).add_(g, alpha=1 - b1) for m, g in zip(s["m"], grads)]
    done = [v.mul_(b2).add_(g * g, alpha=1 - b2) for v, g in zip(s["v"], grads)]
    done = [p.sub_(size * m / (v.sqrt() / root + eps)) for p, m, v in zip(s["params"], s["m"], s["v"])]
    del done
    return {"norm": norm, "p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"]}


def run(state):
    s, c = state, state["case"]
    if own:
        if c["op"] == "attend":
            from diffusion_model_amd.attention import span_attention
            out = span_attention(s["q"], s["k"], s["v"], softcap=c["cap"], slopes=s["slopes"], spans=s["spans"], positions=s["positions"],
                                 causal=c["mask"] == "causal")
            return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])] if c["train"] else [out]
        if c["op"] == "rotate":
            from diffusion_model_amd.embedding import rotary
            q, k = rotary(s["q"], s["k"], s["positions"], s["axes"], interleaved=c["interleaved"])
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))] if c["train"] else [q, k]
        from diffusion_model_amd import optim
        if c["op"] == "clip":
            return {"norm": optim.clip_grad_norm_(s["params"], c["max_norm"]), **s["flat"]}
        s["step"] += 1
        norm = optim.adam_step_(s["params"], s["grads"], s["m"], s["v"], s["step"], lr=2e-4, max_norm=c["max_norm"])
        return {"norm": norm, "p": s["flat_p"], "m": s["flat_m"], "v": s["flat_v"]}
    return {"attend": _plain_attend, "rotate": _plain_rotate, "clip": _plain_clip, "step": _plain_clip}[c["op"]](s)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "attend":
        return _exact_attend(s)
    if c["op"] == "rotate":
        return _exact_rotate(s)
    every = torch.cat([f.double() for f in s["flat"].values()])
    norm = float(torch.linalg.vector_norm(every))
    coef = min(1.0, c["max_norm"] / (norm + 1e-6))
    if c["op"] == "clip":
        return {"norm": torch.tensor(norm, dtype=torch.float64), **{k: f.double() * coef for k, f in s["flat"].items()}}
    t = s["step"] + 1
    g = s["flat"]["fp32"].double() * coef
    m = 0.9 * s["flat_m"].double() + 0.1 * g
    v = 0.999 * s["flat_v"].double() + 0.001 * g ** 2
    p = s["flat_p"].double() - 2e-4 * (m / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)) ** 0.5 + 1e-8)
    # the moments and parameters between the slices are nobody's: they stay
    mine = torch.zeros(g.numel(), dtype=torch.bool, device=g.device)
    for x in s["grads"]:
        o = x.storage_offset()
        mine[o:o + x.numel()] = True
    return {"norm": torch.tensor(norm, dtype=torch.float64), "p": torch.where(mine, p, s["flat_p"].double()),
            "m": torch.where(mine, m, s["flat_m"].double()), "v": torch.where(mine, v, s["flat_v"].double())}


def _exact_attend(s):
    c = s["case"]
    b, nq, nk, h, d = c["batch"], c["nq"], c["nk"], c["heads"], c["dim"]
    if b * h * nq * nk * d * (14 if c["train"] else 4) > 1e14:
        return None
    dev = s["q"].device
    out = torch.zeros(b, nq, h, d, dtype=torch.float64, device=dev)
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(b, nk, c["kv"], d, dtype=torch.float64, device=dev) for _ in range(2))
    key = torch.arange(nk, device=dev)
    for head in range(h):
        shared = head // (h // c["kv"])
        for at in range(0, b, max(1, (1 << 28) // (nq * nk))):           # some samples at a time: 2 GiB an array
            few = slice(at, at + max(1, (1 << 28) // (nq * nk)))
            q, k, v = s["q"][few, :, head].detach().double(), s["k"][few, :, shared].detach().double(), s["v"][few, :, shared].detach().double()
            x = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
            slope = torch.ones_like(x)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
                slope = 1 - (x / c["cap"]) ** 2
            if s["positions"] is not None:
                row = s["positions"][few].long()[..., None]
            else:
                row = (torch.arange(nq, device=dev) + (nk - nq))[None, :, None]
            if s["slopes"] is not None:
                x = x - float(s["slopes"][head]) * torch.abs(key - row).double()
            hidden = torch.zeros_like(x, dtype=torch.bool)
            if s["spans"] is not None:
                first, last = s["spans"][few, :, 0, None], s["spans"][few, :, 1, None]
                hidden |= (key < first) | (key >= last)
            if c["mask"] == "causal":
                hidden |= key > row
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            p = p.masked_fill(hidden, 0.0)                               # a row that sees nothing is nought, not NaN
            del x
            o = torch.bmm(p, v)
            out[few, :, head] = o
            if c["train"]:
                do = s["dout"][few, :, head].double()
                dv[few, :, shared] += torch.bmm(p.transpose(1, 2).contiguous(), do)
                dx = p * (torch.bmm(do, v.transpose(1, 2).contiguous()) - (do * o).sum(-1, keepdim=True)) * slope / math.sqrt(d)
                dq[few, :, head] = torch.bmm(dx, k)
                dk[few, :, shared] += torch.bmm(dx.transpose(1, 2).contiguous(), q)
    return [out, dq, dk, dv] if c["train"] else [out]


def _exact_rotate(s):
    c = s["case"]

    def turned(x, sign):
        y, o = x.detach().double().clone(), 0
        for a, d in enumerate(s["axes"]):
            for i in range(d // 2):
                th = sign * s["positions"][..., a].double() / 10000.0 ** (2 * i / d)
                z = torch.polar(torch.ones_like(th), th)[..., None]
                p, r = (o + 2 * i, o + 2 * i + 1) if c["interleaved"] else (o + i, o + i + d // 2)
                w = torch.complex(x[..., p].detach().double(), x[..., r].detach().double()) * z
                y[..., p], y[..., r] = w.real, w.imag
            o += d
        return y

    out = [turned(s["q"], 1), turned(s["k"], 1)]
    return out + [turned(s["dq"], -1), turned(s["dk"], -1)] if c["train"] else out
