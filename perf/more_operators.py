"""Performance cases of the operators on the condition's way through a served flow batch.

Three operators: rows brought to 8 bits with a scale for each block of 128 (tsplat.fp8.quantize_blocks); a Linear on
such rows and weights, with the step that follows it (tsplat.fp8.fp8_linear); and the cross attention of a batch whose
requests bring encoder states of their own lengths (tsplat.cross_attention.cross_attention).  Inputs follow the flow
model: activations after a norm ~ N(0, 1) with a few large features, weights of a trained Linear's size, queries and
keys after the per-head norm.
"""
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = Path(__file__).resolve().parents[1] / "triposplat-cpu-avx512_amd"
DEV = torch.device("cuda", 0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128
TOP = 448.0  # the largest e4m3 value


def linear(name, rows, k, n, dtype, activation, gated):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "activation": activation,
            "gated": gated}


def quantize(name, rows, k, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "k": k, "dtype": dtype}


def cross(name, queries, keys, heads, kv_heads, dim, dtype, biased):
    return {"name": name, "op": "cross", "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "biased": biased}


def text(lengths):
    return ",".join(str(n) for n in lengths)


def numbers(lengths):
    return [int(n) for n in lengths.split(",")]


def listed():
    return [
        # one camera token through a square Linear: latency alone
        linear("linear_1x1024x1024", 1, 1024, 1024, "fp32", "none", False),
        # the timestep rows of 64 requests through the shared modulation
        linear("linear_64x1024x6144", 64, 1024, 6144, "fp32", "none", False),
        # one request's encoder states to keys and values kept in 16 bits for all steps; a ragged row count
        linear("linear_4101x1024x2048_bf16", 4101, 1024, 2048, "bf16", "none", False),
        # the full latent through fc1 with its GELU
        linear("linear_16384x1024x4096_gelu", 16384, 1024, 4096, "fp32", "gelu", False),
        # the full latent through fc2 onto the gated residual
        linear("linear_16384x4096x1024_gated", 16384, 4096, 1024, "fp32", "none", True),
        # one activation row for several Linears, an odd width
        quantize("quantize_3x1001_fp16", 3, 1001, "fp16"),
        # the MLP's hidden rows of the full latent
        quantize("quantize_16384x4096", 16384, 4096, "fp32"),
        # the camera tokens of a guided pair over their conditions
        cross("cross_2x1_fp32", "1,1", "2049,4101", 16, 16, 64, "fp32", False),
        # one token of each of 64 requests over encoder states kept in bf16, four query heads to a key head
        cross("cross_64x1_gqa_bf16", text([1] * 64), text([128 + 8064 * (i * 37 % 64) // 63 for i in range(64)]),
              32, 8, 128, "bf16", False),
        # the full latent of a guided pair over the benchmark's condition
        cross("cross_2x16384x2048_fp32", "16384,16384", "2048,2048", 16, 16, 64, "fp32", False),
        # requests of several lengths, one of them without a condition, some of the states masked
        cross("cross_ragged_bias_bf16", "4096,8193,1,2049,257", "1370,0,4101,2048,77", 16, 16, 64, "bf16", True),
        # odd heads of 72 values, three query heads to a key head
        cross("cross_3x1001_h6x72_fp16", "1001,513,130", "1025,333,2", 6, 2, 72, "fp16", False),
    ]


def spread(rng, low, high):
    """A whole number between the two, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op, dtype = rng.choice(("linear", "linear", "quantize", "cross", "cross")), rng.choice(("fp32", "bf16", "fp16"))
    if op == "linear":
        k, n = spread(rng, 64, 4096), spread(rng, 16, 6144)
        rows = spread(rng, 1, max(1, min(16384, 60_000_000_000 // (k * n), 60_000_000 // n)))
        c = linear("", rows, k, n, dtype, rng.choice(("none", "none", "gelu")), rng.random() < 0.3)
    elif op == "quantize":
        k = spread(rng, 16, 8192)
        c = quantize("", spread(rng, 1, min(16384, 60_000_000 // k)), k, dtype)
    else:
        kv_heads, dim = rng.randint(1, 16), 8 * rng.randint(2, 16)
        heads = kv_heads * rng.choice((1, 1, 2, 4, 8))
        requests, most_q = rng.randint(1, 24), spread(rng, 1, 16384)
        most_k = spread(rng, 1, min(16384, max(1, 500_000_000 // (requests * heads * most_q)),
                                    max(1, 100_000_000 // (requests * kv_heads * dim))))
        most_q = min(most_q, max(1, 100_000_000 // (requests * heads * dim)))
        queries = [spread(rng, 1, most_q) for _ in range(requests)]
        keys = [spread(rng, 1, most_k) if rng.random() < 0.95 else 0 for _ in range(requests)]
        c = cross("", text(queries), text(keys), heads, kv_heads, dim, dtype, rng.random() < 0.4)
    del c["name"]
    return c


def normal(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device=DEV) * std + mean


def rows_of_a_layer(gen, rows, k, dtype):
    """Activations after a norm and its modulation: some features several times as large as the others."""
    large = 1 + 15 * (torch.rand(k, generator=gen, device=DEV) < 0.02)
    return (normal(gen, rows, k) * large).to(TYPES[dtype])


def prepare_linear(case, gen):
    m, k, n, dtype = (case[key] for key in ("rows", "k", "n", "dtype"))
    s = {"x": rows_of_a_layer(gen, m, k, dtype), "bias": normal(gen, n, std=0.01),
         "activation": None if case["activation"] == "none" else case["activation"], "residual": None, "gate": None}
    w = normal(gen, n, k, std=0.02)
    if case["gated"]:
        s["residual"], s["gate"] = normal(gen, m, n, std=3.0).to(TYPES[dtype]), normal(gen, 1, n, std=0.2)
    if own:  # the packed weight that a program keeps; the plain form keeps the values that it stands for
        from tsplat.fp8 import quantize_blocks

        return s | {"weight": quantize_blocks(w)}
    return s | {"raw": w, "weight": plain_values(*plain_blocks(w), k).t().contiguous()}


def prepare_quantize(case, gen):
    return {"x": rows_of_a_layer(gen, case["rows"], case["k"], case["dtype"])}


def prepare_cross(case, gen):
    queries, keys, heads, kv_heads, d = numbers(case["queries"]), numbers(case["keys"]), *(
        case[key] for key in ("heads", "kv_heads", "dim"))
    dt = TYPES[case["dtype"]]

    def normed(x):
        return x * (math.sqrt(d) / x.norm(dim=-1, keepdim=True))

    tq, tk = sum(queries), sum(keys)
    kv = normal(gen, tk, 2, kv_heads, d)  # rows of the fused projection: k and v are views of them
    kv[:, 0] = normed(kv[:, 0])
    kv = kv.to(dt)
    s = {"q": normed(normal(gen, tq, heads, d)).to(dt), "k": kv[:, 0], "v": kv[:, 1], "bias": None,
         "lengths": (queries, keys)}
    if case["biased"]:  # one state in eight is masked, one stands for a few equal ones
        pick = torch.rand(tk, generator=gen, device=DEV)
        s["bias"] = torch.where(pick < 0.125, -math.inf, torch.where(pick > 0.99, math.log(7.0), 0.0)).to(torch.float32)
    if own:
        from tsplat.cross_attention import CrossPlan

        s["plan"] = CrossPlan(queries, keys, heads, d, kv_heads=kv_heads, dtype=dt, device=DEV)
    else:
        s |= plain_plan(queries, keys)
    return s


def plain_plan(queries, keys):
    """Where each request's rows lie in a batch padded to the longest: row numbers (0 past a request's end), and which of
    them are real."""
    s = {}
    for name, lengths in (("q", queries), ("k", keys)):
        n = torch.tensor(lengths, device=DEV)
        at = torch.arange(max(max(lengths), 1), device=DEV)
        real = at < n[:, None]
        s[name + "_real"] = real
        s[name + "_rows"] = torch.where(real, at + (n.cumsum(0) - n)[:, None], 0)
    return s


def prepare(case, seed):
    if own and str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"linear": prepare_linear, "quantize": prepare_quantize, "cross": prepare_cross}[case["op"]](case, gen)
    return s | {"op": case["op"]}


# ------------------------------------------------------------------ the framework's calls
def run_own(s):
    if s["op"] == "linear":
        from tsplat.fp8 import fp8_linear

        return fp8_linear(s["x"], s["weight"], s["bias"], activation=s["activation"], gate=s["gate"],
                          residual=s["residual"])
    if s["op"] == "quantize":
        from tsplat.fp8 import quantize_blocks

        q = quantize_blocks(s["x"])
        return q.codes, q.exponents
    from tsplat.cross_attention import cross_attention

    return cross_attention(s["q"], s["k"], s["v"], s["plan"], key_bias=s["bias"])


# ------------------------------------------------------------------ the plain forms
def plain_blocks(x):
    """x [M, K] -> (e4m3 codes [M, blocks, 128], the exponent of each block's scale + 127).  The scale is the smallest
    power of two that brings the block's largest value to 448 or below: exact in any type."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)  # top = part * 2^power, part in [1/2, 1); 448 = 0.875 * 2^9
    e = power - 9 + (part > 0.875).to(power.dtype)
    e = torch.where(top > 0, e.clamp(-127, 127), 0)
    return (x * power_of_two(-e)[:, :, None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def power_of_two(e):
    """2^e by its bits: pow() is a step off here and there, which moves values next to a border."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64).float()


def plain_values(codes, exponents, k):
    return (codes.float() * power_of_two(exponents.to(torch.int32) - 127)[:, :, None]).flatten(1)[:, :k]


def plain_linear(s):
    y = plain_values(*plain_blocks(s["x"]), s["x"].shape[1]) @ s["weight"] + s["bias"]
    if s["activation"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    y = y if s["gate"] is None else y * s["gate"]
    y = y if s["residual"] is None else y + s["residual"].float()
    return y.to(s["x"].dtype)


def plain_quantize(s):
    codes, exponents = plain_blocks(s["x"])
    return codes.flatten(1)[:, :s["x"].shape[1]], exponents


def plain_cross(s):
    """The batch padded to its longest request; key heads' query heads are rows of one product."""
    (tq, heads, d), kv_heads = s["q"].shape, s["k"].shape[1]
    if s["k"].shape[0] == 0:
        return torch.zeros_like(s["q"])
    r, lq = s["q_rows"].shape
    lk, group = s["k_rows"].shape[1], heads // kv_heads
    q = (s["q"].float() / math.sqrt(d))[s["q_rows"]].view(r, lq, kv_heads, group, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float()[s["k_rows"]].permute(0, 2, 3, 1).contiguous()
    v = s["v"].float()[s["k_rows"]].transpose(1, 2).contiguous()
    scores = torch.matmul(q.reshape(r, kv_heads, group * lq, d), k)
    add = torch.where(s["k_real"], 0.0 if s["bias"] is None else s["bias"][s["k_rows"]], -math.inf)
    scores += add[:, None, None]
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top > -math.inf, top, 0.0)
    scores.exp_()
    out = torch.matmul(scores, v) / scores.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.view(r, kv_heads, group, lq, d).permute(0, 3, 1, 2, 4).reshape(r, lq, heads, d)
    return out[s["q_real"]].to(s["q"].dtype)


def run(state):
    if own:
        return run_own(state)
    return {"linear": plain_linear, "quantize": plain_quantize, "cross": plain_cross}[state["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact_blocks(x):
    """(code values, scales, scale exponents + 127) in 64 bits: borders by comparison, rounding by the spacing of e4m3."""
    m, k = x.shape
    x = torch.cat((x.double(), torch.zeros(m, -k % BLOCK, dtype=torch.float64, device=DEV)), 1).view(m, -1, BLOCK)
    power = torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64, device=DEV)
    top = x.abs().max(-1).values
    at = torch.searchsorted(TOP * power, top)  # the first scale that 448 of reach the largest value
    scale = power[torch.where(top == 0, 160, at.clamp(33, 287))]
    v = x / scale[:, :, None]
    least = v.abs().clamp_min(2.0 ** -6)
    step = power[torch.searchsorted(power, least, right=True) - 1] / 8
    return (v / step).round() * step, scale, torch.where(top == 0, 127, at.clamp(33, 287) - 33).to(torch.uint8)


def exact_values(x):
    v, scale, _ = exact_blocks(x)
    return (v * scale[:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous()


def exact_linear(s):
    y = exact_values(s["x"]) @ exact_values(s["raw"]).t().contiguous() + s["bias"].double()
    if s["activation"] == "gelu":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if s["gate"] is not None:
        y = y * s["gate"].double()
    return y if s["residual"] is None else y + s["residual"].double()


def exact_quantize(s):
    v, _, e = exact_blocks(s["x"])
    return v.reshape(len(v), -1)[:, :s["x"].shape[1]], e


def exact_cross(s):
    (tq, heads, d), kv_heads = s["q"].shape, s["k"].shape[1]
    out = torch.zeros(tq, heads, d, dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for nq, nk in zip(*s["lengths"]):
        if nq and nk:
            q = s["q"][q0:q0 + nq].double().transpose(0, 1)
            k, v = (s[key][k0:k0 + nk].double().transpose(0, 1).repeat_interleave(heads // kv_heads, 0).contiguous()
                    for key in ("k", "v"))
            t = torch.bmm(q.contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(d)
            if s["bias"] is not None:
                t = t + s["bias"][k0:k0 + nk].double()
            out[q0:q0 + nq] = torch.bmm(torch.softmax(t, -1).nan_to_num(0.0), v).transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": exact_linear, "quantize": exact_quantize, "cross": exact_cross}[case["op"]](s)


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case.get("dtype")]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": size * m * (k + n * (2 if case["gated"] else 1)) + n * (k + k // BLOCK + 4),
                "flops": 2 * m * n * k}
    if case["op"] == "quantize":
        m, k = case["rows"], case["k"]
        return {"bytes": m * (size * k + k + -(-k // BLOCK)), "flops": 3 * m * k}
    queries, keys = numbers(case["queries"]), numbers(case["keys"])
    pairs = sum(a * b for a, b in zip(queries, keys))
    rows = 2 * sum(queries) * case["heads"] + 2 * sum(keys) * case["kv_heads"]
    return {"bytes": size * rows * case["dim"] + (4 * sum(keys) if case["biased"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}
