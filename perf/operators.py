"""Performance cases of the operators that one block of a served flow batch runs besides its packed products.

Three operators: the low-rank adapters of a batch's requests added to a shared projection
(tsplat.adapters.low_rank_add); a branch's output normed, gated and added to the residual stream, with the next
norm and its modulation (tsplat.block_ops.residual_norm); and rotary positions of several axes with the per-head
RMSNorm, written in the attention's layout (tsplat.qkv.rope_axes, qkv_rope_axes).  Inputs follow the flow model:
activations after a norm ~ N(0, 1), a residual stream of a few units, adapters as a fine-tune leaves them.
"""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = Path(__file__).resolve().parents[1] / "triposplat-cpu-avx512_amd"
DEV = torch.device("cuda", 0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
HEAD_EPS = 1e-12
THETA = 10000.0


def adapt(name, rows, k, n, rank, slots, requests, dtype):
    return {"name": name, "op": "adapt", "rows": rows, "k": k, "n": n, "rank": rank, "slots": slots,
            "requests": requests, "dtype": dtype}


def norm(name, batch, length, c, pre, post, affine, gate, modulate):
    return {"name": name, "op": "norm", "batch": batch, "length": length, "c": c, "pre": pre, "post": post,
            "affine": affine, "gate": gate, "modulate": modulate}


def rope(name, form, batch, length, heads, dim, axes, interleaved, fractional, far):
    return {"name": name, "op": "rope", "form": form, "batch": batch, "length": length, "heads": heads, "dim": dim,
            "axes": axes, "interleaved": interleaved, "fractional": fractional, "far": far}


def listed():
    return [
        # the camera token's rows of a guided pair through one adapted square Linear: latency alone
        adapt("adapt_2x1024x1024_r16", 2, 1024, 1024, 16, 4, 2, "bf16"),
        # the timestep rows of 64 requests through the shared modulation, each with an adapter of its own
        adapt("adapt_64x1024x6144_r32", 64, 1024, 6144, 32, 64, 64, "fp16"),
        # three requests of the reference model's length, ragged, through fc1; one of them has no adapter
        adapt("adapt_12294x1024x4096_r16", 12294, 1024, 4096, 16, 4, 3, "bf16"),
        # the full latent of one request and its guided twin through fc2, adapters kept in 32 bits
        adapt("adapt_16384x4096x1024_r64", 16384, 4096, 1024, 64, 2, 2, "fp32"),
        # one camera token of a guided pair
        norm("norm_2x1x1024", 2, 1, 1024, "layer", "none", False, True, True),
        # the reference model's length after attention: gated residual, LayerNorm, the MLP's modulation
        norm("norm_1x12294x1024", 1, 12294, 1024, "layer", "none", False, True, True),
        # norms before and after the branch, of a wide residual stream, no gate
        norm("norm_2x4101x4096_sandwich", 2, 4101, 4096, "rms", "rms", True, False, False),
        # an odd width
        norm("norm_3x1001x1023", 3, 1001, 1023, "layer", "layer", True, True, False),
        # one token's q against a long cache of positions
        rope("rope_q_2x1x16x64", "q", 2, 1, 16, 64, 3, True, False, 1000003),
        # q, k and v of the full latent, time x height x width
        rope("rope_qkv_16384x16x64", "qkv", 1, 16384, 16, 64, 3, True, False, 0),
        # image tokens at fractional places (another resolution than trained), halves paired, larger heads
        rope("rope_qkv_2x4101x8x128_half", "qkv", 2, 4101, 8, 128, 2, False, True, 0),
        # a guided pair's condition keys, odd heads of 72 values
        rope("rope_q_2x2049x7x72", "q", 2, 2049, 7, 72, 2, True, False, 4096),
    ]


def spread(rng, low, high):
    """A whole number between the two, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("adapt", "norm", "rope"))
    if op == "adapt":
        k, n, rank, slots = spread(rng, 64, 4096), spread(rng, 64, 6144), spread(rng, 1, 128), spread(rng, 1, 64)
        most = min(16384, 100_000_000 // (k + 2 * n), 10_000_000_000 // (rank * slots * (k + n)))
        rows = spread(rng, 1, max(1, most))
        c = adapt("", rows, k, n, rank, slots, spread(rng, 1, min(rows, 256)), rng.choice(("fp32", "bf16", "fp16")))
    elif op == "norm":
        width = spread(rng, 32, 8192)
        length = spread(rng, 1, max(1, 33_000_000 // (4 * width)))
        c = norm("", rng.randint(1, 4), length, width, rng.choice(("layer", "rms")),
                 rng.choice(("none", "layer", "rms")), rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.7)
    else:
        axes, heads, batch = rng.randint(1, 3), rng.randint(1, 24), rng.randint(1, 3)
        dim = 2 * rng.randint(max(8, axes), 128)
        length = spread(rng, 1, max(1, 16_000_000 // (batch * heads * dim)))
        c = rope("", rng.choice(("q", "qkv")), batch, length, heads, dim, axes, rng.random() < 0.5,
                 rng.random() < 0.5, rng.choice((0, 0, 4096, 1000003)))
    del c["name"]
    return c


def pieces(total, parts):
    """`total` in `parts` of about equal size, the first ones longer."""
    return [total // parts + (i < total % parts) for i in range(parts)]


def normal(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device=DEV) * std + mean


def request_slots(case, gen):
    """The slot of each row: requests of ragged lengths in a row, about one in five of them without an adapter
    (-1); every slot has its turn where there are enough requests."""
    m, q, slots = case["rows"], case["requests"], case["slots"]
    if q < m:
        cuts = torch.sort(torch.randperm(m - 1, generator=gen, device=DEV)[:q - 1] + 1).values
    else:
        cuts = torch.arange(1, m, device=DEV)
    place = torch.zeros(m, dtype=torch.int64, device=DEV)
    place[cuts] = 1
    of_request = torch.randperm(max(q, slots), generator=gen, device=DEV)[:q] % slots
    bare = torch.rand(q, generator=gen, device=DEV) < 0.2
    bare[0] = False
    return torch.where(bare, -1, of_request)[place.cumsum(0)].to(torch.int32)


def slot_ranks(case):
    """Fine-tunes of several ranks."""
    return [max(1, case["rank"] - (i % 4) * (case["rank"] // 4)) for i in range(case["slots"])]


def prepare_adapt(case, gen):
    m, k, n, r, slots = (case[key] for key in ("rows", "k", "n", "rank", "slots"))
    dt = TYPES[case["dtype"]]
    ranks = slot_ranks(case)
    live = torch.arange(r, device=DEV) < torch.tensor(ranks, device=DEV)[:, None]
    down = (normal(gen, slots, r, k, std=1 / math.sqrt(k)) * live[:, :, None]).to(dt)
    up = (normal(gen, slots, n, r, std=1 / math.sqrt(r)) * live[:, None, :]).to(dt)
    s = {"x": normal(gen, m, k), "y": normal(gen, m, n), "down": down, "up": up,
         "scale": torch.rand(slots, generator=gen, device=DEV) + 0.5, "slots": request_slots(case, gen)}
    if own:
        from tsplat.adapters import AdapterBank

        s["bank"] = AdapterBank.stack(down, up, s["scale"], ranks)
    return s


def prepare_norm(case, gen):
    b, length, c = case["batch"], case["length"], case["c"]
    s = {"x": normal(gen, b, length, c, std=3.0, mean=0.5), "h": normal(gen, b, length, c),
         "residual_scale": 1.0 if case["gate"] else 0.75, "pre": case["pre"], "post": case["post"]}
    weights = ("weight", "post_weight") if case["affine"] else ()
    s |= {key: normal(gen, c, std=0.05, mean=1.0) if key in weights else None for key in ("weight", "post_weight")}
    for key, kind in (("bias", "pre"), ("post_bias", "post")):
        s[key] = normal(gen, c, std=0.02) if case["affine"] and case[kind] == "layer" else None
    if case["post"] == "none":
        s["post_weight"] = None
    mod = normal(gen, b, 3 * c, std=0.2)  # one row a request, as the modulation Linear leaves it
    s["gate"] = mod[:, :c] if case["gate"] else None
    s["scale"], s["shift"] = (mod[:, c:2 * c], mod[:, 2 * c:]) if case["modulate"] else (None, None)
    return s


def prepare_rope(case, gen):
    b, length, heads, d, axes = (case[key] for key in ("batch", "length", "heads", "dim", "axes"))
    side = max(1, round(length ** (1 / axes)))
    place = torch.arange(length, device=DEV)
    grid = torch.stack([place // side ** (axes - 1 - i) % (side if i else length + 1) for i in range(axes)], -1)
    start = torch.randint(0, 64, (b, 1, axes), generator=gen, device=DEV)
    start[:, :, 0] += case["far"]
    at = grid + start
    parts = 3 if case["form"] == "qkv" else 1
    return {"x": normal(gen, b * length, parts * heads * d), "b": b, "l": length, "h": heads, "d": d,
            "positions": (at.float() * 0.8125 if case["fractional"] else at.to(torch.int32)).contiguous(),
            "sections": pieces(d // 2, axes), "interleaved": case["interleaved"], "form": case["form"],
            "gamma": normal(gen, parts, heads, d, std=0.05, mean=1.0)} | rope_plan(d, axes, case["interleaved"])


def rope_plan(d, axes, interleaved):
    if not own:
        return {}
    from tsplat.qkv import RopeAxes

    return {"rope": RopeAxes(d, pieces(d // 2, axes), THETA, interleaved=interleaved, device=DEV)}


def prepare(case, seed):
    if own and str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"adapt": prepare_adapt, "norm": prepare_norm, "rope": prepare_rope}[case["op"]](case, gen)
    return s | {"op": case["op"]}


# ------------------------------------------------------------------ the framework's calls
def run_own(s):
    if s["op"] == "adapt":
        from tsplat.adapters import low_rank_add

        return low_rank_add(s["y"], s["x"], s["bank"], s["slots"])
    if s["op"] == "norm":
        from tsplat.block_ops import residual_norm

        return residual_norm(s["x"], s["h"], gate=s["gate"], residual_scale=s["residual_scale"],
                             post_norm=None if s["post"] == "none" else s["post"], post_weight=s["post_weight"],
                             post_bias=s["post_bias"], post_eps=EPS, norm=s["pre"], weight=s["weight"],
                             bias=s["bias"], eps=EPS, scale=s["scale"], shift=s["shift"])
    if s["form"] == "q":
        from tsplat.qkv import rope_axes

        return rope_axes(s["x"].view(s["b"], s["l"], s["h"], s["d"]), s["positions"], s["rope"], gamma=s["gamma"][0],
                         eps=HEAD_EPS)
    from tsplat.qkv import qkv_rope_axes

    return qkv_rope_axes(s["x"], s["positions"], s["rope"], s["gamma"][0], s["gamma"][1], s["b"], s["l"], s["h"],
                         eps=HEAD_EPS)


# ------------------------------------------------------------------ the plain forms
def plain_adapt(s):
    """Every row through every slot's adapter in two products, what is not its own taken to zero between them."""
    down, up = s["down"].float(), s["up"].float()
    slots, r, k = down.shape
    t = s["x"] @ down.reshape(slots * r, k).t()
    slot_of_column = torch.arange(slots * r, device=DEV) // r
    t = torch.where(s["slots"][:, None] == slot_of_column, t * s["scale"][slot_of_column], 0.0)
    return s["y"] + t @ up.transpose(1, 2).reshape(slots * r, -1)


def plain_one_norm(x, kind, weight, bias):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    x = x if weight is None else x * weight
    return x if bias is None else x + bias


def plain_norm(s):
    h = plain_one_norm(s["h"], s["post"], s["post_weight"], s["post_bias"])
    h = h if s["gate"] is None else h * s["gate"][:, None]
    x = s["x"] * s["residual_scale"] + h
    y = plain_one_norm(x, s["pre"], s["weight"], s["bias"])
    return x, y if s["scale"] is None else y * (1 + s["scale"][:, None]) + s["shift"][:, None]


def plain_rope(s):
    b, length, heads, d = s["b"], s["l"], s["h"], s["d"]
    axis = torch.tensor([i for i, n in enumerate(s["sections"]) for _ in range(n)], device=DEV)
    ramp = torch.tensor([THETA ** (-j / n) for n in s["sections"] for j in range(n)], dtype=torch.float64, device=DEV)
    angle = s["positions"].double()[:, :, axis] * ramp
    cos, sin = angle.cos().float()[:, :, None, :], angle.sin().float()[:, :, None, :]

    def rotated(x, gamma):
        pair = x.view(b, length, heads, d // 2, 2) if s["interleaved"] else x.view(b, length, heads, 2, d // 2).transpose(3, 4)
        re, im = pair[..., 0], pair[..., 1]
        turned = torch.stack((re * cos - im * sin, re * sin + im * cos), -1 if s["interleaved"] else -2)
        turned = turned.reshape(b, length, heads, d)
        size = torch.sqrt((turned * turned).sum(-1, keepdim=True)).clamp_min(HEAD_EPS)
        return (turned * (math.sqrt(d) / size) * gamma).transpose(1, 2).contiguous()

    if s["form"] == "q":
        return rotated(s["x"], s["gamma"][0])
    q, k, v = s["x"].view(b, length, 3, heads, d).unbind(2)
    return (rotated(q.contiguous(), s["gamma"][0]), rotated(k.contiguous(), s["gamma"][1]),
            v.transpose(1, 2).contiguous())


def run(state):
    if own:
        return run_own(state)
    return {"adapt": plain_adapt, "norm": plain_norm, "rope": plain_rope}[state["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact_adapt(s):
    out = s["y"].double()
    for a in range(len(s["scale"])):
        at = torch.nonzero(s["slots"] == a)[:, 0]
        if len(at):
            inner = s["x"][at].double() @ s["down"][a].double().t().contiguous()
            out[at] += s["scale"][a].double() * (inner @ s["up"][a].double().t().contiguous())
    return out


def exact_norm(s):
    def of(v, kind, weight, bias):
        if kind == "layer":
            v = (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + EPS)
        elif kind == "rms":
            v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
        v = v * weight.double() if weight is not None else v
        return v + bias.double() if bias is not None else v

    h = of(s["h"].double(), s["post"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        h = h * s["gate"].double().unsqueeze(1)
    x = s["residual_scale"] * s["x"].double() + h
    y = of(x, s["pre"], s["weight"], s["bias"])
    if s["scale"] is not None:
        y = y + y * s["scale"].double().unsqueeze(1) + s["shift"].double().unsqueeze(1)
    return x, y


def exact_rope(s):
    b, length, heads, d = s["b"], s["l"], s["h"], s["d"]
    turns, first = [], 0
    for i, n in enumerate(s["sections"]):
        f = torch.tensor([THETA ** (-j / n) for j in range(n)], dtype=torch.float64, device=DEV)
        turns.append(s["positions"][:, :, i:i + 1].double() * f)
        first += n
    spin = torch.polar(torch.ones(b, length, first, dtype=torch.float64, device=DEV), torch.cat(turns, -1))[:, None]

    def of(x, gamma):
        x = x.double().reshape(b, length, heads, d).transpose(1, 2)
        if s["interleaved"]:
            z = torch.view_as_real(torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) * spin).flatten(-2)
        else:
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * spin
            z = torch.cat((z.real, z.imag), -1)
        return z * math.sqrt(d) / z.norm(dim=-1, keepdim=True).clamp_min(HEAD_EPS) * gamma.double()[:, None]

    w = heads * d
    if s["form"] == "q":
        return of(s["x"], s["gamma"][0])
    v = s["x"][:, 2 * w:].double().reshape(b, length, heads, d).transpose(1, 2).contiguous()
    return of(s["x"][:, :w], s["gamma"][0]), of(s["x"][:, w:2 * w], s["gamma"][1]), v


def exact(case, seed):
    s = prepare(case, seed)
    return {"adapt": exact_adapt, "norm": exact_norm, "rope": exact_rope}[case["op"]](s)


def work(case):
    if case["op"] == "adapt":
        m, k, n, used = case["rows"], case["k"], case["n"], min(case["slots"], case["requests"])
        r = sum(slot_ranks(case)) / case["slots"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 4 * m * (k + 2 * n + 1) + size * used * r * (k + n), "flops": 2 * m * r * (k + n)}
    if case["op"] == "norm":
        m, c = case["batch"] * case["length"], case["c"]
        return {"bytes": 16 * m * c, "flops": 20 * m * c}
    tokens, parts = case["batch"] * case["length"], 3 if case["form"] == "qkv" else 1
    values = tokens * case["heads"] * case["dim"] * parts
    return {"bytes": 8 * values + 4 * tokens * case["axes"], "flops": 6 * values}
