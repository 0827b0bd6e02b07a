"""The gradients of a mixture-of-experts layer that this file measures: those of the experts' products, and checkpoints of activations
in 8 bits with their use in the backward pass.

A case is one of four kinds.

  dgrad       moe_dgrad: the gradient of the rows that went into the experts' products, rows times weights across their rows
  wgrad       moe_wgrad: the gradient of the experts' weights, a sum over each expert's own rows, in the weights' type or in fp32 as
              optimisers keep it; with `checkpoint` the products' input is there in 8 bits only
  checkpoint  moe_checkpoint: rows to 8 bits; where `gated`, moe_swiglu_checkpoint: the gated activation between the experts' two
              products, and its input in 8 bits from the same read
  backward    moe_swiglu_backward: the gradient of the activation's input, and the activation's output again for the second product's
              weights; from 16 bits, or from the checkpoint

Checkpoint: a block of 32 values of a row (of either half of a gated row; the last one may be shorter) shares a scale 2^(b - 127), b the least
byte with which the largest magnitude is at most 448 times the scale; a code is the e4m3 number nearest to the value over the scale, ties to the even one, and
values beyond 15/8 times the type's largest power of two count as that much.

Token counts run from a few dozen to a whole training batch.  Activations are N(0, 1) with a few outlier channels, weights N(0, 0.02),
gradients N(0, 0.01), routing the top-k of N(0, 1) logits, uniform, or Zipf with exponent 1.2.  Where `dropped` is not 0, that share of
the pairs exceeds its expert's capacity: the rows behind the last routed one belong to no expert.
"""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LARGEST = {"bf16": 1.875 * 2.0**127, "f16": 1.875 * 2.0**15}
BLOCK = 32


def _product(name, kind, dtype, tokens, topk, experts, hidden, ffn, routing="softmax", dropped=0.0, out=None, checkpoint=False):
    case = {"name": name, "kind": kind, "dtype": dtype, "tokens": tokens, "topk": topk, "experts": experts, "hidden": hidden, "ffn": ffn,
            "routing": routing, "dropped": dropped}
    if kind == "wgrad":
        case.update(out=out or dtype, checkpoint=checkpoint)
    return case


def _rows(name, kind, dtype, rows, cols, gated=False, checkpoint=False):
    case = {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "cols": cols}
    case.update({"gated": gated} if kind == "checkpoint" else {"checkpoint": checkpoint})
    return case


def listed():
    return [
        # A few sequences' last tokens in fine-tuning, eight large experts: their weights are read for a handful of rows each.
        _product("dgrad_few_bf16", "dgrad", "bf16", 37, 2, 8, 4096, 14336),
        # A whole training batch over eight large experts.
        _product("dgrad_train_bf16", "dgrad", "bf16", 8192, 2, 8, 4096, 14336),
        # A training batch over many small experts with a skewed load, a capacity and dropped pairs, in fp16.
        _product("dgrad_fine_f16", "dgrad", "f16", 16384, 6, 64, 2048, 1408, "zipf", dropped=0.05),
        # The same batches' weight gradients: in the weights' own type ...
        _product("wgrad_train_bf16", "wgrad", "bf16", 8192, 2, 8, 4096, 14336),
        # ... and in fp32, for an optimiser that sums several batches, at widths that are no whole tiles.
        _product("wgrad_fine_f16", "wgrad", "f16", 16384, 6, 64, 2040, 1400, "zipf", dropped=0.05, out="f32"),
        # A wide layer of many experts whose input was kept in 8 bits.
        _product("wgrad_wide_8bit_bf16", "wgrad", "bf16", 4096, 8, 32, 7168, 2048, "uniform", out="f32", checkpoint=True),
        # A small layer and batch, its input kept in 8 bits: fewer tiles than compute units.
        _product("wgrad_small_8bit_bf16", "wgrad", "bf16", 256, 2, 8, 1024, 2048, checkpoint=True),
        # The input of a layer's first products, kept in 8 bits.
        _rows("checkpoint_bf16", "checkpoint", "bf16", 16384, 4096),
        # The activation of a whole training batch, and its input in 8 bits.
        _rows("swiglu_train_bf16", "checkpoint", "bf16", 16384, 14336, gated=True),
        # That of a few tokens in fp16, at a width that no block divides.
        _rows("swiglu_few_f16", "checkpoint", "f16", 74, 1407, gated=True),
        # Backwards from the 8 bits.
        _rows("swiglu_grad_8bit_bf16", "backward", "bf16", 16384, 14336, checkpoint=True),
        # Backwards from 16 bits, a microbatch in fp16.
        _rows("swiglu_grad_f16", "backward", "f16", 1000, 1408),
    ]


# ---- inputs ---------------------------------------------------------------------------------------------------


def _choose_experts(routing, tokens, topk, experts, gen):
    if routing == "softmax":
        return torch.topk(torch.randn(tokens, experts, generator=gen, device="cuda"), topk, dim=-1).indices
    logp = torch.zeros(experts, device="cuda")  # without replacement from a fixed distribution: the top-k of log p + Gumbel noise
    if routing == "zipf":
        logp = -1.2 * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    u = torch.rand(tokens, experts, generator=gen, device="cuda").clamp_(1e-9, 1 - 1e-7)
    return torch.topk(logp - torch.log(-torch.log(u)), topk, dim=-1).indices


def _splits(case, gen):
    """Rows of each expert."""
    flat = _choose_experts(case["routing"], case["tokens"], case["topk"], case["experts"], gen).flatten()
    if case["dropped"] > 0:
        lost = torch.rand(flat.numel(), generator=gen, device="cuda") < case["dropped"]
        flat = torch.where(lost, case["experts"], flat)
    return torch.bincount(flat, minlength=case["experts"] + 1)[: case["experts"]].to(torch.int32)


def _activations(rows, cols, dtype, gen):
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::97] *= 8.0  # a few outlier channels, as activations have them
    return x.to(DTYPES[dtype])


def _gradients(rows, cols, dtype, gen):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * 0.01).to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, s = case["dtype"], {"case": case}
    if case["kind"] in ("dgrad", "wgrad"):
        rows, k, n, e = case["tokens"] * case["topk"], case["hidden"], case["ffn"], case["experts"]
        s["splits"] = _splits(case, gen)
        s["splits_host"] = s["splits"].tolist()
        s["grad"] = _gradients(rows, n, dtype, gen)
        if case["kind"] == "dgrad":
            s["weight"] = torch.empty(e, n, k, dtype=DTYPES[dtype], device="cuda")
            for i in range(e):
                s["weight"][i] = torch.randn(n, k, generator=gen, device="cuda") * 0.02
            return s
        s["input"], s["scale"] = _activations(rows, k, dtype, gen), None
        if case["checkpoint"]:
            s["input"], s["scale"] = _checkpoint(s["input"], dtype)
        return s
    rows, cols = case["rows"], case["cols"]
    s["x"], s["scale"] = _activations(rows, cols * 2 if case["kind"] == "backward" or case["gated"] else cols, dtype, gen), None
    if case["kind"] == "backward":
        s["grad"] = _gradients(rows, cols, dtype, gen)
        if case["checkpoint"]:
            s["x"], s["scale"] = _checkpoint_halves(s["x"], dtype)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------


def _power(byte):
    """2^(byte - 127), exactly; 255 is NaN."""
    byte = byte.to(torch.int32)
    power = torch.where(byte == 0, 1 << 22, byte << 23).view(torch.float32)
    return torch.where(byte == 255, math.nan, power)


def _checkpoint(x, dtype):
    """x [rows, cols] -> codes in e4m3 [rows, cols] and scales in e8m0 [rows, ceil(cols / 32)].  All steps but the code's rounding are exact."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    bits = x.abs().amax(-1).view(torch.int32)  # the pattern of the largest magnitude: exponent, and whether it is over 1.75 times its power of two
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0)
    byte = torch.where(bits >> 23 == 255, 255, byte)
    down = ((254 - byte.clamp(max=253)) << 23).view(torch.float32).unsqueeze(-1)
    codes = x.clamp(-LARGEST[dtype], LARGEST[dtype]) * down
    codes = torch.where((byte == 255).unsqueeze(-1), 0.0, codes).view(rows, -1)[:, :cols]
    return codes.to(torch.float8_e4m3fn).contiguous(), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _checkpoint_halves(x, dtype):
    """Both halves of a gated row in blocks of their own."""
    f = x.shape[1] // 2
    (gate, gate_scale), (up, up_scale) = _checkpoint(x[:, :f], dtype), _checkpoint(x[:, f:], dtype)
    return torch.cat([gate.view(torch.uint8), up.view(torch.uint8)], 1).view(torch.float8_e4m3fn), torch.cat(
        [gate_scale.view(torch.uint8), up_scale.view(torch.uint8)], 1).view(torch.float8_e8m0fnu)


def _values(codes, scale):
    return codes.float() * _power(scale.view(torch.uint8)).repeat_interleave(BLOCK, 1)[:, : codes.shape[1]]


def _halves(x, scale):
    """The gate and up values, in fp32."""
    f = x.shape[1] // 2
    if scale is None:
        return x[:, :f].float(), x[:, f:].float()
    kb = scale.shape[1] // 2
    return _values(x[:, :f], scale[:, :kb]), _values(x[:, f:], scale[:, kb:])


def _sorted_out(codes, scale):
    return {"codes": codes, "scale": scale.view(torch.uint8)}


def _plain(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    if case["kind"] == "dgrad":
        rest = s["grad"].shape[0] - sum(s["splits_host"])
        by_expert = s["grad"].split(s["splits_host"] + [rest])
        return {"grad_input": torch.cat([(g.float() @ w.float()).to(dtype) for g, w in zip(by_expert, s["weight"])] + [by_expert[-1].new_zeros(rest, case["hidden"])])}
    if case["kind"] == "wgrad":
        rows = sum(s["splits_host"])
        x = (s["input"][:rows].float() if s["scale"] is None else _values(s["input"][:rows], s["scale"][:rows])).split(s["splits_host"])
        return {"grad_weight": torch.stack([(g.float().t() @ v).to(DTYPES[case["out"]]) for g, v in zip(s["grad"][:rows].split(s["splits_host"]), x)])}
    if case["kind"] == "checkpoint" and not case["gated"]:
        return _sorted_out(*_checkpoint(s["x"], case["dtype"]))
    gate, up = _halves(s["x"], s["scale"])
    sig = torch.sigmoid(gate)
    out = {"out": (gate * sig * up).to(dtype)}
    if case["kind"] == "checkpoint":
        return {**out, **_sorted_out(*_checkpoint_halves(s["x"], case["dtype"]))}
    grad = s["grad"].float()
    d_gate, d_up = grad * up * sig * (1 + gate * (1 - sig)), grad * gate * sig
    return {**out, "grad_input": torch.cat([d_gate.to(dtype), d_up.to(dtype)], 1)}


# ---- the framework's operators -----------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _flux():
    import flux_amd

    return flux_amd


def _own(s):
    case, flux = s["case"], _flux()
    if case["kind"] == "dgrad":
        return {"grad_input": flux.moe_dgrad(s["grad"], s["weight"], s["splits"])}
    if case["kind"] == "wgrad":
        return {"grad_weight": flux.moe_wgrad(s["grad"], s["input"], s["splits"], input_scale=s["scale"], output_dtype=DTYPES[case["out"]])}
    if case["kind"] == "backward":
        grad_input, out = flux.moe_swiglu_backward(s["grad"], s["x"], s["scale"])
        return {"out": out, "grad_input": grad_input}
    if not case["gated"]:
        return _sorted_out(*flux.moe_checkpoint(s["x"]))
    out, codes, scale = flux.moe_swiglu_checkpoint(s["x"])
    return {"out": out, **_sorted_out(codes, scale)}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------


def _two_to(e):
    """2^e in 64 bits for whole e, from its pattern: a library's power may be off in the last bit, which breaks ties."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_checkpoint(x, dtype):
    """Codes' values and scale bytes of x [rows, cols]: the scale by logarithm, the code as the nearest on the grid of e4m3."""
    rows, cols = x.shape
    blocks = torch.cat([x.double(), x.new_zeros(rows, -cols % 32, dtype=torch.float64)], 1).view(rows, -1, 32)
    most = blocks.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(most > 0, most, 2.0**-200) / 448.0))
    e = e - (_two_to(e - 1) * 448 >= most).double() + (_two_to(e) * 448 < most).double()
    e = e.clamp(min=-127)
    a = blocks.abs().clamp(max=LARGEST[dtype]) / _two_to(e)
    step = _two_to(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
    step = torch.where(a >= step * 16, step * 2, torch.where((a < step * 8) & (step > 2.0**-9), step / 2, step))
    low = torch.floor(a / step)
    rest = a / step - low
    low = low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 == 1))).double()
    codes = torch.sign(blocks) * low * step
    return codes.view(rows, -1)[:, :cols], (e.squeeze(2) + 127).to(torch.uint8)


def _exact_values(codes, scale):
    byte = scale.view(torch.uint8).double()
    return codes.double() * _two_to(byte - 127).repeat_interleave(32, dim=1)[:, : codes.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("dgrad", "wgrad"):
        at, out = 0, []
        for e, rows in enumerate(s["splits_host"]):
            mine = slice(at, at + rows)
            grad = s["grad"][mine].double()
            if case["kind"] == "dgrad":
                out.append(grad @ s["weight"][e].double())
            else:
                x = s["input"][mine].double() if s["scale"] is None else _exact_values(s["input"][mine], s["scale"][mine])
                out.append(grad.t() @ x)
            at += rows
        if case["kind"] == "wgrad":
            return {"grad_weight": torch.stack(out)}
        return {"grad_input": torch.cat(out + [torch.zeros(s["grad"].shape[0] - at, case["hidden"], dtype=torch.float64, device="cuda")])}
    x, f = s["x"], case["cols"]
    if case["kind"] == "checkpoint" and not case["gated"]:
        codes, scale = _exact_checkpoint(x, case["dtype"])
        return {"codes": codes, "scale": scale}
    if s["scale"] is None:
        gate, up = x[:, :f].double(), x[:, f:].double()
    else:
        kb = s["scale"].shape[1] // 2
        gate, up = _exact_values(x[:, :f], s["scale"][:, :kb]), _exact_values(x[:, f:], s["scale"][:, kb:])
    silu = gate / (1 + torch.exp(-gate))
    if case["kind"] == "checkpoint":
        parts = [_exact_checkpoint(half, case["dtype"]) for half in (x[:, :f], x[:, f:])]
        return {"out": silu * up, "codes": torch.cat([p[0] for p in parts], 1), "scale": torch.cat([p[1] for p in parts], 1)}
    grad, e = s["grad"].double(), torch.exp(-gate)
    slope = (1 + e + gate * e) / (1 + e).square()  # of silu
    return {"out": silu * up, "grad_input": torch.cat([grad * up * slope, grad * silu], 1)}


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _experts_hit(case):
    """Expected number of experts with at least one row."""
    t, k, e = case["tokens"], case["topk"], case["experts"]
    if case["routing"] == "zipf":
        p = [(i + 1) ** -1.2 for i in range(e)]
        share = [min(1.0, k * v / sum(p)) for v in p]
    else:
        share = [k / e] * e
    return sum(1.0 - (1.0 - s) ** t for s in share)


def work(case):
    """Inputs read once, outputs written once; of weights those of the experts that are hit."""
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["kind"] in ("dgrad", "wgrad"):
        m = case["tokens"] * case["topk"]
        routed, k, n = round(m * (1 - case["dropped"])), case["hidden"], case["ffn"]
        if case["kind"] == "dgrad":
            bytes_ = 2 * routed * n + 2 * int(_experts_hit(case) * n * k) + 2 * m * k
        else:
            x = routed * (k + -(-k // BLOCK)) if case["checkpoint"] else 2 * routed * k
            bytes_ = 2 * routed * n + x + case["experts"] * n * k * size[case["out"]]
        return {"bytes": bytes_, "flops": 2 * routed * k * n}
    rows, cols = case["rows"], case["cols"]
    kept = rows * (cols + -(-cols // BLOCK))  # codes and scales of one half
    if case["kind"] == "checkpoint":
        if not case["gated"]:
            return {"bytes": 2 * rows * cols + kept, "flops": 0}
        return {"bytes": 6 * rows * cols + 2 * kept, "flops": 0}
    return {"bytes": 8 * rows * cols + (2 * kept if case["checkpoint"] else 4 * rows * cols), "flops": 0}


# ---- drawn cases ------------------------------------------------------------------------------------------------


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(["dgrad", "wgrad", "checkpoint", "backward"], [4, 5, 3, 3])[0]
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind in ("checkpoint", "backward"):
        cols = 32 * _log_int(rng, 2, 448)
        if rng.random() < 0.3:
            cols -= rng.randint(1, 31)
        case = {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, 32768), "cols": cols}
        case["gated" if kind == "checkpoint" else "checkpoint"] = rng.random() < 0.6
        return case
    topk = rng.choice([1, 2, 2, 4, 6, 8])
    case = {"kind": kind, "dtype": dtype, "tokens": _log_int(rng, 16, 16384), "topk": topk, "experts": _log_int(rng, max(4, topk), 96),
            "hidden": 128 * _log_int(rng, 4, 64), "ffn": 128 * _log_int(rng, 4, 112), "routing": rng.choice(["softmax", "uniform", "zipf"]),
            "dropped": rng.choice([0.0, 0.0, 0.05])}
    if rng.random() < 0.3:  # widths that are no whole tiles
        case["hidden"] -= 8 * rng.randint(1, 15)
        case["ffn"] -= 8 * rng.randint(1, 15)
    if rng.random() < 0.1:  # nor whole vectors
        case["hidden"] -= rng.randint(1, 7)
        case["ffn"] -= rng.randint(1, 7)
    if kind == "wgrad":
        case.update(out=rng.choice([dtype, "f32"]), checkpoint=rng.random() < 0.5)
    return case


def draw(rng):
    """One more case of the same ranges: no more bytes or arithmetic than the largest listed one."""
    largest = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in largest), max(w["flops"] for w in largest)
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= bytes_ and w["flops"] <= flops and case.get("experts", 1) * case.get("ffn", 0) * case.get("hidden", 0) <= 6e8:
            return case
