"""Measured cases of the image-token attention operators: qkv_norm_rope, block_select and block_attention.

``run`` computes each operator in plain torch where ``own`` is false and through the package's public entry points
where it is true; ``exact`` gives the operators' definition in 64 bits. Sizes follow the shipped UNet (latents of
64 x 64 with 8 heads of 40 channels, two guidance branches, batches of 8), the same network's 1024 x 1024 images and
short videos, with single tokens and odd grids at the ends of the range.
"""
import importlib
import math

import torch

own = False

BLOCK_Q = 128  # query rows that share one selection
THETA = 10000.0
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One query token's heads, e.g. a class or register token appended to a running grid: launch latency.
        dict(name="rope one token", op="rope", n=1, frames=1, height=1, width=1, heads=8, kv_heads=8, dim=40,
             axis_t=0, axis_h=20, axis_w=20, pairing="adjacent", norm=True, x_type="f32", out_type="f32", far=0),
        # The first UNet level of eight guided inpaints: f32 projections into half-precision attention operands.
        dict(name="rope unet level 0", op="rope", n=16, frames=1, height=64, width=64, heads=8, kv_heads=8, dim=40,
             axis_t=0, axis_h=20, axis_w=20, pairing="halves", norm=True, x_type="f32", out_type="f16", far=0),
        # A batch of odd crops with fewer key heads, part of each head left unrotated.
        dict(name="rope odd crops", op="rope", n=3, frames=1, height=37, width=53, heads=10, kv_heads=5, dim=80,
             axis_t=0, axis_h=32, axis_w=32, pairing="adjacent", norm=True, x_type="f32", out_type="bf16", far=5000),
        # A 16-frame video of 1024 x 1024 windows (64 x 64 tokens after patching): the streaming rate.
        dict(name="rope video", op="rope", n=1, frames=16, height=64, width=64, heads=16, kv_heads=8, dim=128,
             axis_t=16, axis_h=56, axis_w=56, pairing="adjacent", norm=True, x_type="bf16", out_type="bf16", far=0),
        # Selection for the first UNet level of eight guided inpaints.
        dict(name="select unet level 0", op="select", n=16, nq=4096, nk=4096, heads=8, kv_heads=8, dim=40,
             block_k=64, topk=16, type="f16", mask="none"),
        # Odd crops whose masked-out pixels must not steer the choice.
        dict(name="select masked crops", op="select", n=2, nq=1961, nk=4133, heads=10, kv_heads=5, dim=80,
             block_k=32, topk=24, type="f32", mask="hole"),
        # Selection over a 16-frame video: many query blocks against many key blocks.
        dict(name="select video", op="select", n=1, nq=65536, nk=65536, heads=16, kv_heads=8, dim=128,
             block_k=64, topk=64, type="bf16", mask="none"),
        # One new token against a long video's keys: latency, and the split over the listed blocks.
        dict(name="attend one token", op="attend", n=1, nq=1, nk=65536, heads=16, kv_heads=8, dim=128,
             block_k=64, topk=64, type="bf16", mask="none"),
        # The first UNet level of eight guided inpaints in the engine's own precision.
        dict(name="attend unet level 0", op="attend", n=16, nq=4096, nk=4096, heads=8, kv_heads=8, dim=40,
             block_k=64, topk=16, type="f32", mask="none"),
        # Odd crops with a hole in the keys, narrow blocks, fewer key heads.
        dict(name="attend masked crops", op="attend", n=2, nq=1961, nk=4133, heads=10, kv_heads=5, dim=80,
             block_k=32, topk=24, type="f32", mask="hole"),
        # Two 1024 x 1024 images' latents, half precision, wide blocks.
        dict(name="attend 1024 px", op="attend", n=2, nq=16384, nk=16384, heads=16, kv_heads=16, dim=64,
             block_k=128, topk=16, type="f16", mask="none"),
        # An 8-frame video: the compute rate.
        dict(name="attend video", op="attend", n=1, nq=32768, nk=32768, heads=16, kv_heads=8, dim=128,
             block_k=64, topk=32, type="bf16", mask="none"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "select", "attend"])
    n = _log_int(rng, 1, 16)
    heads, kv_heads = rng.choice([(8, 8), (16, 8), (10, 5), (16, 16), (12, 12), (6, 1), (1, 1)])
    dim = rng.choice([40, 64, 80, 128, 8 * rng.randint(2, 16)])
    if op == "rope":
        frames = rng.choice([1, 1, 1, _log_int(rng, 2, 16)])
        height, width = _log_int(rng, 1, 96), _log_int(rng, 1, 96)
        row = (heads + 2 * kv_heads) * dim
        frames = max(1, min(frames, 130_000_000 // (height * width * row)))
        n = max(1, min(n, 130_000_000 // (frames * height * width * row)))
        pairs = dim // 2
        axis_t = 2 * rng.randint(0, pairs // 4) if frames > 1 else 0
        axis_h = 2 * rng.randint(1, (pairs - axis_t // 2) // 2)
        axis_w = rng.choice([axis_h, dim - axis_t - axis_h])
        x_type, out_type = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                                       ("bf16", "bf16")])
        return dict(op=op, n=n, frames=frames, height=height, width=width, heads=heads, kv_heads=kv_heads, dim=dim,
                    axis_t=axis_t, axis_h=axis_h, axis_w=axis_w, pairing=rng.choice(["adjacent", "halves"]),
                    norm=rng.random() < 0.8, x_type=x_type, out_type=out_type, far=rng.choice([0, 5000, 1_000_000]))
    type_, block_k = rng.choice(["f32", "f16", "bf16"]), rng.choice([16, 32, 64, 128])
    row = dim * (4 if type_ == "f32" else 2)
    if op == "select":  # enough blocks and heads for a choice to depend on the inputs
        heads, kv_heads = (8, 4) if heads < 8 else (heads, kv_heads)
        nk = _log_int(rng, 9 * block_k, 32768)
        nq = rng.choice([nk, nk, _log_int(rng, 1, 32768), 1])
        topk = _log_int(rng, 1, min(nk // block_k // 2, 4096 // block_k))
        n = max(1, min(n, 400_000_000 // (row * (heads * nq + kv_heads * nk))))
    else:
        nk = _log_int(rng, 1, 32768)
        nq = rng.choice([nk, nk, _log_int(rng, 1, 32768), 1])
        topk = _log_int(rng, 1, max(1, min(-(-nk // block_k) + 2, 4096 // block_k)))
        n = max(1, min(n, 400_000_000 // (2 * row * (heads * nq + kv_heads * nk))))
        pairs = 2.7e11 / 2 / (topk * block_k * dim * heads)
        n = max(1, min(n, int(pairs // max(nq, BLOCK_Q))))
        nq = max(1, min(nq, int(pairs // n)))
    mask = rng.choice(["none", "none", "hole", "length", "empty" if n > 1 else "length"])
    return dict(op=op, n=n, nq=nq, nk=nk, heads=heads, kv_heads=kv_heads, dim=dim, block_k=block_k, topk=topk,
                type=type_, mask=mask)


def work(case):
    c = case
    if c["op"] == "rope":
        tokens = c["n"] * c["frames"] * c["height"] * c["width"]
        values = tokens * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        size = {"f32": 4, "f16": 2, "bf16": 2}
        return {"bytes": values * (size[c["x_type"]] + size[c["out_type"]]) + tokens // c["n"] * 12,
                "flops": 8 * tokens * (c["heads"] + c["kv_heads"]) * c["dim"]}
    size = 4 if c["type"] == "f32" else 2
    q_blocks, k_blocks = -(-c["nq"] // BLOCK_Q), -(-c["nk"] // c["block_k"])
    topk = min(c["topk"], k_blocks)
    mask = c["n"] * c["nk"] if c["mask"] != "none" else 0
    q_bytes = c["n"] * c["nq"] * c["heads"] * c["dim"] * size
    if c["op"] == "select":
        k_bytes = c["n"] * c["nk"] * c["kv_heads"] * c["dim"] * size
        return {"bytes": q_bytes + k_bytes + mask + 4 * c["n"] * c["heads"] * q_blocks * c["topk"],
                "flops": 2 * c["n"] * c["heads"] * q_blocks * k_blocks * c["dim"]
                + c["n"] * (c["nq"] * c["heads"] + c["nk"] * c["kv_heads"]) * c["dim"]}
    # Of the keys and values, no more than the listed blocks can be needed, each at most once.
    keys = min(c["nk"], topk * c["block_k"])
    rows = c["n"] * min(c["kv_heads"] * c["nk"], c["heads"] * q_blocks * keys)
    return {"bytes": 2 * q_bytes + 2 * rows * c["dim"] * size + mask + 4 * c["n"] * c["heads"] * q_blocks * c["topk"],
            "flops": 4 * c["n"] * c["heads"] * c["nq"] * keys * c["dim"]}


# ------------------------------------------------------------------------------------------------- inputs

def _field(gen, n, tokens, heads, dim, run):
    """Neighbouring tokens resemble each other: a coarse random field, stretched, plus independent noise."""
    coarse = torch.randn(n, tokens // run + 2, heads, dim, generator=gen, device="cuda")
    x = coarse.repeat_interleave(run, dim=1)[:, 13:13 + tokens] if run > 13 else coarse[:, :tokens]
    return x + 0.7 * torch.randn(n, tokens, heads, dim, generator=gen, device="cuda")


def _mask(c, gen):
    """[n, nk] bytes, 1 where a key may be attended to; None without a mask."""
    if c["mask"] == "none":
        return None
    n, nk = c["n"], c["nk"]
    m = torch.ones(n, nk, dtype=torch.uint8, device="cuda")
    at = torch.arange(nk, device="cuda")[None]
    if c["mask"] == "hole":  # an inpainting hole: a run of keys, and some stray ones
        start = torch.randint(0, nk, (n, 1), generator=gen, device="cuda") // 2
        m[(at >= start) & (at < start + nk // 3)] = 0
        m[torch.rand(n, nk, generator=gen, device="cuda") < 0.05] = 0
    else:  # a padded batch; "empty" leaves the last item without any key
        length = torch.randint(nk // 2, nk + 1, (n, 1), generator=gen, device="cuda")
        m[at >= length] = 0
        if c["mask"] == "empty":
            m[-1] = 0
    return m


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda").manual_seed(seed)
    if c["op"] == "rope":
        tokens = c["frames"] * c["height"] * c["width"]
        heads, kv, dim, out = c["heads"], c["kv_heads"], c["dim"], TYPES[c["out_type"]]
        x = _field(gen, c["n"], tokens, heads + 2 * kv, dim, 17) * 1.5
        grid = torch.meshgrid(*(torch.arange(c[s], device="cuda") for s in ("frames", "height", "width")),
                              indexing="ij")
        start = torch.randint(0, c["far"] + 1, (3,), generator=gen, device="cuda")  # the window's place in the image
        return dict(
            case=c, x=x.reshape(c["n"], tokens, -1).to(TYPES[c["x_type"]]),
            positions=torch.stack([g.reshape(-1) for g in grid], -1).add(start).float().contiguous(),
            q_gamma=1 + 0.1 * torch.randn(dim, generator=gen, device="cuda"),
            k_gamma=1 + 0.1 * torch.randn(dim, generator=gen, device="cuda"),
            q=torch.empty(c["n"], tokens, heads, dim, dtype=out, device="cuda"),
            k=torch.empty(c["n"], tokens, kv, dim, dtype=out, device="cuda"),
            v=torch.empty(c["n"], tokens, kv, dim, dtype=out, device="cuda"))
    kind = TYPES[c["type"]]
    s = dict(case=c, q=_field(gen, c["n"], c["nq"], c["heads"], c["dim"], 150).to(kind),
             k=_field(gen, c["n"], c["nk"], c["kv_heads"], c["dim"], 70).to(kind), mask=_mask(c, gen))
    if c["op"] == "attend":
        s["v"] = _field(gen, c["n"], c["nk"], c["kv_heads"], c["dim"], 40).to(kind)
        s["out"] = torch.empty_like(s["q"])
        s["index"] = _plain_select(s)
    else:
        s["index"] = torch.empty(c["n"], c["heads"], -(-c["nq"] // BLOCK_Q), c["topk"], dtype=torch.int32,
                                 device="cuda")
    if s["mask"] is not None:  # what a mask hides may hold anything
        s["k"][s["mask"] == 0] = float("nan")
        if "v" in s:
            s["v"][s["mask"] == 0] = float("inf")
    return s


# ------------------------------------------------------------------------------------------------- plain forms

def _plain_rotate(x, angles, offset, size, pairing):
    """Rotates channels [offset, offset + size) of x [n, tokens, heads, dim] by angles [tokens, size / 2]."""
    cos, sin = angles.cos().float()[None, :, None], angles.sin().float()[None, :, None]
    part = x[..., offset:offset + size]
    if pairing == "adjacent":
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :size // 2], part[..., size // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([x[..., :offset], turned, x[..., offset + size:]], -1)


def _plain_head(x, gamma, s):
    c = s["case"]
    x = x.float()
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma
    offset = 0
    for axis, size in enumerate((c["axis_t"], c["axis_h"], c["axis_w"])):
        if size:
            steps = torch.arange(size // 2, device="cuda", dtype=torch.float64)
            angles = s["positions"][:, axis, None].double() * THETA ** (-2.0 * steps / size)
            x = _plain_rotate(x, angles, offset, size, c["pairing"])
        offset += size
    return x


def _plain_rope(s):
    c, out = s["case"], TYPES[s["case"]["out_type"]]
    x = s["x"].unflatten(-1, (-1, c["dim"]))
    q, k, v = x.split([c["heads"], c["kv_heads"], c["kv_heads"]], 2)
    return _plain_head(q, s["q_gamma"], s).to(out), _plain_head(k, s["k_gamma"], s).to(out), v.to(out)


def _blocks(x, size):
    """[n, tokens, ...] -> [n, blocks, size, ...], the last block filled up with zeros."""
    short = -x.shape[1] % size
    if short:
        x = torch.cat([x, x.new_zeros(x.shape[0], short, *x.shape[2:])], 1)
    return x.unflatten(1, (-1, size))


def _plain_select(s):
    """A block's score is the mean query's product with the mean unmasked key, in 64 bits since scores lie close."""
    c, q, k = s["case"], s["q"].double(), s["k"].double()
    keep = torch.ones(c["n"], c["nk"], device="cuda") if s["mask"] is None else s["mask"]
    keep = keep.double()[..., None, None]
    count = _blocks(keep, c["block_k"]).sum(2)
    k_mean = _blocks(torch.where(keep > 0, k, 0.0), c["block_k"]).sum(2) / count.clamp(min=1)
    q_mean = _blocks(q, BLOCK_Q).sum(2) / _blocks(torch.ones_like(q[:, :, :1, :1]), BLOCK_Q).sum(2)
    k_mean = k_mean.repeat_interleave(c["heads"] // c["kv_heads"], 2)
    score = q_mean.permute(0, 2, 1, 3) @ k_mean.permute(0, 2, 3, 1)  # [n, heads, q blocks, k blocks]
    some = (count[..., 0, 0] > 0)[:, None, None, :].expand_as(score)
    order = score.masked_fill(~some, -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :c["topk"]]
    none = 1 << 30
    order = order.masked_fill(~some.gather(-1, order), none).sort(-1).values
    order = torch.nn.functional.pad(order, (0, c["topk"] - order.shape[-1]), value=none)
    return order.masked_fill(order == none, -1).int()


def _plain_attend(s):
    c, group = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    rows = min(BLOCK_Q, c["nq"])
    keep = torch.ones(c["n"], c["nk"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"] > 0
    live = keep[..., None, None]
    q = _blocks(s["q"].float(), rows).permute(0, 3, 1, 2, 4)  # [n, heads, q blocks, rows, dim]
    k = _blocks(torch.where(live, s["k"], 0.0).float(), c["block_k"])
    v = _blocks(torch.where(live, s["v"], 0.0).float(), c["block_k"])
    index = s["index"].long()
    item = torch.arange(c["n"], device="cuda")[:, None, None, None]
    head = (torch.arange(c["heads"], device="cuda") // group)[None, :, None, None]
    at = index.clamp(min=0)
    k, v = (t.permute(0, 3, 1, 2, 4)[item, head, at].flatten(3, 4) for t in (k, v))  # [..., topk * block_k, dim]
    open_ = (_blocks(keep, c["block_k"])[item, at] & (index >= 0)[..., None]).flatten(3)[..., None, :]
    score = (q @ k.transpose(-1, -2) / math.sqrt(c["dim"])).masked_fill(~open_, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :c["nq"]].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- one pass

_context = None


def _views(s):
    """The package's handles of the state's tensors and the workspace, made once as a user's program keeps them."""
    global _context
    mbx = importlib.import_module("moebius-cpu_b200")
    if _context is None:
        _context = mbx.Context(0)
        _context.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream's handle
    kinds = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: mbx.bfloat16, torch.int32: "int32",
             torch.uint8: "uint8"}
    t = {k: mbx.DeviceTensor.wrap(_context, x.data_ptr(), x.shape, dtype=kinds[x.dtype])
         for k, x in s.items() if isinstance(x, torch.Tensor)}
    c = s["case"]
    if c["op"] == "select":
        t["workspace"] = mbx.block_select_workspace(t["q"], t["k"], block_k=c["block_k"])
    elif c["op"] == "attend":
        t["workspace"] = mbx.block_attention_workspace(t["q"], t["k"], t["index"], block_k=c["block_k"])
    return mbx, t


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "select": _plain_select, "attend": _plain_attend}[c["op"]](s)
    if "views" not in s:
        s["views"] = _views(s)
    mbx, t = s["views"]
    if c["op"] == "rope":
        mbx.qkv_norm_rope(t["x"], c["heads"], c["kv_heads"], c["dim"], positions=t["positions"],
                          axis_dims=(c["axis_t"], c["axis_h"], c["axis_w"]), theta=THETA, pairing=c["pairing"],
                          norm=c["norm"], q_gamma=t["q_gamma"], k_gamma=t["k_gamma"], eps=EPS,
                          out=(t["q"], t["k"], t["v"]))
        return s["q"], s["k"], s["v"]
    if c["op"] == "select":
        mbx.block_select(t["q"], t["k"], c["topk"], block_k=c["block_k"], key_mask=t.get("mask"),
                         workspace=t["workspace"], out=t["index"])
        return s["index"]
    mbx.block_attention(t["q"], t["k"], t["v"], t["index"], block_k=c["block_k"], key_mask=t.get("mask"),
                        workspace=t["workspace"], out=t["out"])
    return s["out"]


# ------------------------------------------------------------------------------------------------- 64 bits

def _exact_rope(s):
    c = s["case"]
    x = s["x"].double().reshape(c["n"], -1, c["heads"] + 2 * c["kv_heads"], c["dim"])
    cut = (c["heads"], c["heads"] + c["kv_heads"])
    done = []
    for part, gamma in ((x[:, :, :cut[0]], s["q_gamma"]), (x[:, :, cut[0]:cut[1]], s["k_gamma"])):
        y = part.clone()
        if c["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() * gamma.double()
        first = 0
        for axis, size in enumerate((c["axis_t"], c["axis_h"], c["axis_w"])):
            half = size // 2
            for i in range(half):
                a, b = (first + 2 * i, first + 2 * i + 1) if c["pairing"] == "adjacent" else (first + i,
                                                                                              first + half + i)
                turn = s["positions"][:, axis].double() * math.exp(-math.log(THETA) * 2 * i / size)
                z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(turn), turn)[None, :, None]
                y[..., a], y[..., b] = z.real, z.imag
            first += size
        done.append(y)
    return done[0], done[1], x[:, :, cut[1]:]


def _exact_select(s):
    c = s["case"]
    q_blocks, k_blocks = -(-c["nq"] // BLOCK_Q), -(-c["nk"] // c["block_k"])
    q, k = s["q"].double(), s["k"].double()
    found = torch.full((c["n"], c["heads"], q_blocks, c["topk"]), -1, dtype=torch.int32, device="cuda")
    means, some = [], []
    for j in range(k_blocks):
        part = k[:, j * c["block_k"]:(j + 1) * c["block_k"]]
        m = torch.ones_like(part[..., 0, 0]) if s["mask"] is None else s["mask"][:, j * c["block_k"]:
                                                                                 (j + 1) * c["block_k"]].double()
        means.append(torch.einsum("nb,nbhd->nhd", m, torch.where(m[..., None, None] > 0, part, 0.0))
                     / m.sum(1).clamp(min=1)[:, None, None])
        some.append(m.sum(1) > 0)
    means, some = torch.stack(means, 1), torch.stack(some, 1)
    for i in range(q_blocks):
        mean = q[:, i * BLOCK_Q:(i + 1) * BLOCK_Q].mean(1)
        for h in range(c["heads"]):
            score = torch.einsum("nd,njd->nj", mean[:, h], means[:, :, h * c["kv_heads"] // c["heads"]])
            score = score.masked_fill(~some, -math.inf)
            best = torch.argsort(-score, dim=1, stable=True)[:, :c["topk"]]
            best = best.masked_fill(~some.gather(1, best), k_blocks).sort(1).values.int()
            found[:, h, i, :best.shape[1]] = torch.where(best == k_blocks, -1, best)
    return found


def _exact_attend(s):
    c = s["case"]
    k_blocks = -(-c["nk"] // c["block_k"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(c["n"]):
        live = torch.ones(c["nk"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][i] > 0
        for h in range(c["heads"]):
            kh = h * c["kv_heads"] // c["heads"]
            k, v = s["k"][i, live, kh].double(), s["v"][i, live, kh].double()
            listed_ = s["index"][i, h].long()
            chosen = torch.zeros(listed_.shape[0], k_blocks + 1, dtype=torch.bool, device="cuda")
            chosen.scatter_(1, listed_.masked_fill(listed_ < 0, k_blocks), True)
            chosen = chosen[:, :k_blocks].repeat_interleave(c["block_k"], 1)[:, :c["nk"]][:, live]
            for start in range(0, c["nq"], 64 * BLOCK_Q):
                q = s["q"][i, start:start + 64 * BLOCK_Q, h].double()
                here = chosen[start // BLOCK_Q:start // BLOCK_Q + 64].repeat_interleave(BLOCK_Q, 0)[:q.shape[0]]
                logit = torch.where(here, (q @ k.T) * c["dim"] ** -0.5, -math.inf)
                out[i, start:start + 64 * BLOCK_Q, h] = torch.nan_to_num(torch.softmax(logit, 1), nan=0.0) @ v
    return out


def exact(case, seed):
    if case["op"] == "attend" and case["n"] * case["heads"] * case["nq"] * case["nk"] > 3e10:
        return None
    return {"rope": _exact_rope, "select": _exact_select, "attend": _exact_attend}[case["op"]](prepare(case, seed))
