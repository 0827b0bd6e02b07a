"""The operators of a mixture-of-experts layer that this file measures: tokens sorted by expert and back with their gradients,
and 4-bit microscaled floating point (MXFP4) with the experts' products on it.

A case is one of four kinds.

  permute    moe_permute: every token's row copied to the rows of its experts; or its backward pass, the sum of a
             token's gradient rows
  unpermute  moe_unpermute: the experts' rows back in token order, summed with the router's weights; or its backward
             pass, the gradients of the rows and of the weights
  quant      a tensor to MXFP4 and back to the values that its codes stand for, along the rows and, for a backward
             pass, along the columns as well
  product    activations quantised to MXFP4, then multiplied with the MXFP4 weights of their experts (experts = 0: of
             one dense layer), with the rows gathered on the way in or weighted on the way out

MXFP4: blocks of 32 values share a scale 2^(b - 127), b = max(floor(log2 of the largest magnitude) - 2 + 127, 0); a value is the nearest
of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, ties to the even code, and what lies past 6 is 6.  Codes are packed two to a byte, the
lower half first; a row's last block is filled up with zeros.

Token counts run from one token being decoded to a whole prefill batch.  Activations are N(0, 1) with a few outlier
channels, weights N(0, 0.02), routing the top-k of N(0, 1) logits, uniform, or Zipf with exponent 1.2.  Where `dropped`
is not 0, that share of the pairs exceeds its expert's capacity: they have no row (index -1) and the rows behind the last
routed one are zeros.
"""
import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32


def _moe(name, kind, direction, dtype, tokens, topk, experts, hidden, routing="softmax", dropped=0.0):
    case = {"name": name, "kind": kind, "direction": direction, "dtype": dtype, "tokens": tokens, "topk": topk,
            "experts": experts, "hidden": hidden, "routing": routing, "dropped": dropped}
    if kind == "unpermute":
        case["weights"] = "f32"
    return case


def _product(name, dtype, out, tokens, topk, experts, hidden, ffn, routing="softmax", gathered=True, weighted=False):
    return {"name": name, "kind": "product", "dtype": dtype, "out": out, "tokens": tokens, "topk": topk, "experts": experts,
            "hidden": hidden, "ffn": ffn, "routing": routing, "gathered": gathered, "weighted": weighted}


def listed():
    return [
        # A small decode batch sorted by expert: the launch is most of it.
        _moe("permute_decode_bf16", "permute", "forward", "bf16", 37, 2, 8, 4096),
        # A whole prefill batch over many small experts with a skewed load.
        _moe("permute_prefill_bf16", "permute", "forward", "bf16", 16384, 6, 64, 2048, "zipf"),
        # The same step of a training batch backwards, where experts have a capacity and some pairs were dropped.
        _moe("permute_grad_bf16", "permute", "backward", "bf16", 8192, 2, 8, 4096, dropped=0.05),
        # A chunk of a prefill back in token order, in fp16, at a width that no vector divides.
        _moe("unpermute_chunk_f16", "unpermute", "forward", "f16", 777, 8, 32, 2047, "uniform"),
        # A training batch of a wide layer backwards: gradients of the experts' rows and of the router's weights.
        _moe("unpermute_grad_bf16", "unpermute", "backward", "bf16", 4096, 8, 32, 7168, "uniform"),
        # A small training batch in fp32 with dropped pairs.
        _moe("unpermute_grad_f32", "unpermute", "backward", "f32", 1000, 4, 16, 1536, dropped=0.1),
        # The activations of a decode batch.
        {"name": "quant_decode_bf16", "kind": "quant", "dtype": "bf16", "rows": 128, "cols": 7168, "transposed": False},
        # Activations of a training step quantised for forward and backward (both directions from one tensor).
        {"name": "quant_train_bf16", "kind": "quant", "dtype": "bf16", "rows": 11000, "cols": 7168, "transposed": True},
        # One user decoding one token with eight large experts: two experts' weights are read for one row each.
        _product("product_one_bf16", "bf16", "bf16", 1, 2, 8, 4096, 14336),
        # Decoding, one GPU's share of a wide layer: every expert is hit by a few dozen rows.
        _product("product_decode_bf16", "bf16", "bf16", 128, 8, 32, 7168, 2048, "uniform"),
        # A chunk of a prefill between the two regimes, the second product of a layer in fp16: rows already sorted, and
        # weighted on the way out.
        _product("product_chunk_f16", "f16", "f32", 777, 2, 8, 14336, 4096, gathered=False, weighted=True),
        # A whole prefill batch over eight large experts.
        _product("product_prefill_bf16", "bf16", "bf16", 8192, 2, 8, 4096, 14336),
    ]


# ---- inputs ---------------------------------------------------------------------------------------------------


def _choose_experts(routing, tokens, topk, experts, gen):
    """[tokens, topk] expert ids and fp32 weights that sum to one."""
    logits = torch.randn(tokens, experts, generator=gen, device="cuda")
    if routing == "softmax":
        weight, idx = torch.topk(torch.softmax(logits, dim=-1), topk, dim=-1)
    else:  # without replacement from a fixed distribution: the top-k of log p + Gumbel noise
        logp = torch.zeros(experts, device="cuda")
        if routing == "zipf":
            logp = -1.2 * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
        u = torch.rand(tokens, experts, generator=gen, device="cuda").clamp_(1e-9, 1 - 1e-7)
        idx = torch.topk(logp - torch.log(-torch.log(u)), topk, dim=-1).indices
        weight = torch.softmax(torch.gather(logits, 1, idx), dim=-1)
    return idx, weight / weight.sum(dim=-1, keepdim=True)


def _route(case, gen):
    """The stable sort by expert: scatter_index [tokens, topk] (-1: dropped), splits, and by sorted row the token and weight."""
    tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
    chosen, weight = _choose_experts(case["routing"], tokens, topk, experts, gen)
    flat = chosen.flatten()
    if case.get("dropped", 0.0) > 0:
        lost = torch.rand(flat.numel(), generator=gen, device="cuda") < case["dropped"]
        flat = torch.where(lost, experts, flat)
    order = torch.argsort(flat, stable=True)
    scatter = torch.empty_like(order)
    scatter[order] = torch.arange(order.numel(), device="cuda")
    scatter = torch.where(flat == experts, -1, scatter)
    splits = torch.bincount(flat, minlength=experts + 1)[:experts]
    return {"scatter": scatter.to(torch.int32).view(tokens, topk), "splits": splits.to(torch.int32), "splits_host": splits.tolist(),
            "weight": weight, "gather": (order // topk).to(torch.int32), "row_weight": weight.flatten()[order].contiguous()}


def _activations(rows, cols, dtype, gen):
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::97] *= 8.0  # a few outlier channels, as activations have them
    return x.to(DTYPES[dtype])


def _prepare_moe(case, gen):
    t, k, h = case["tokens"], case["topk"], case["hidden"]
    s = _route(case, gen)
    rows, cols = (t, h) if (case["kind"] == "permute") == (case["direction"] == "forward") else (t * k, h)
    s["x"] = _activations(rows, cols, case["dtype"], gen)
    if case["kind"] == "unpermute":
        s["weight"] = s["weight"].to(DTYPES[case["weights"]])
        if case["direction"] == "backward":
            s["grad"], s["x"] = s["x"], _activations(t * k, h, case["dtype"], gen)
    return s


def _prepare_quant(case, gen):
    return {"x": _activations(case["rows"], case["cols"], case["dtype"], gen)}


def _prepare_product(case, gen):
    t, k, e, h, f = (case[n] for n in ("tokens", "topk", "experts", "hidden", "ffn"))
    s = _route(case, gen) if e else {}
    s["x"] = _activations(t * k if e and not case["gathered"] else t, h, case["dtype"], gen)
    kb = -(-h // BLOCK)
    s["w"] = torch.empty(max(e, 1), f, kb * BLOCK // 2, dtype=torch.uint8, device="cuda")
    s["w_scale"] = torch.empty(max(e, 1), f, kb, dtype=torch.uint8, device="cuda")
    for i in range(max(e, 1)):
        value, scale = _quantise(torch.randn(f, h, generator=gen, device="cuda") * 0.02)
        s["w"][i], s["w_scale"][i] = _pack(value), scale
    s["w"] = s["w"].view(torch.float4_e2m1fn_x2)
    s["w_scale"] = s["w_scale"].view(torch.float8_e8m0fnu)
    if not e:
        s["w"], s["w_scale"] = s["w"][0], s["w_scale"][0]
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"permute": _prepare_moe, "unpermute": _prepare_moe, "quant": _prepare_quant, "product": _prepare_product}[case["kind"]]
    return {"case": case, **make(case, gen)}


# ---- the plain forms -------------------------------------------------------------------------------------------


def _float_bits(bits):
    return bits.to(torch.int32).view(torch.float32)


def _quantise(x):
    """x [..., K] -> the codes' values over the scale [..., ceil(K / 32), 32] in fp32 and the scale's byte.  All steps are exact:
    the exponent is read from the bits, and the scale is a power of two."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    exponent = x.abs().amax(-1).view(torch.int32) >> 23
    byte = torch.where(exponent == 255, 255, (exponent - 2).clamp(min=0))
    x = x * _float_bits((254 - byte.clamp(max=253)) << 23).unsqueeze(-1)
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    return torch.copysign(a, x), byte.to(torch.uint8)


def _scale_of(byte):
    byte = byte.to(torch.int32)
    power = _float_bits(torch.where(byte == 0, 1 << 22, byte << 23))
    return torch.where(byte == 255, math.nan, power)


def _values(value, byte):
    return (value * _scale_of(byte).unsqueeze(-1)).flatten(-2)


def _pack(value):
    """The packed codes of values that lie on the grid."""
    a = value.abs()
    code = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, 7.0)).to(torch.uint8) | (torch.signbit(value).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4)


@functools.lru_cache(maxsize=None)
def _pairs():
    """[256, 2]: the two values of every byte."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    grid = torch.cat([grid, -grid])
    byte = torch.arange(256, device="cuda")
    return torch.stack([grid[byte & 15], grid[byte >> 4]], dim=1)


def _unpack(codes, scale):
    value = _pairs()[codes.view(torch.uint8).int()].flatten(-2).unflatten(-1, (-1, BLOCK))
    return _values(value, scale.view(torch.uint8))


def _rows_of(scatter, rows):
    """Row of each pair, with one more row for those that have none."""
    return torch.where(scatter < 0, rows, scatter).flatten().long()


def _plain_moe(s):
    case, scatter, x = s["case"], s["scatter"], s["x"]
    tokens, topk = scatter.shape
    rows, h = tokens * topk, x.shape[1]
    at = _rows_of(scatter, rows)

    def to_rows(per_pair):  # [tokens, topk, h] in the order of the rows
        out = torch.zeros(rows + 1, h, dtype=x.dtype, device=x.device)
        out[at] = per_pair.reshape(rows, h).to(x.dtype)
        return out[:rows]

    def to_pairs(by_row):
        return torch.cat([by_row, by_row.new_zeros(1, h)])[at].float().view(tokens, topk, h)

    if case["kind"] == "permute":
        if case["direction"] == "forward":
            return {"rows": to_rows(x.unsqueeze(1).expand(tokens, topk, h))}
        return {"grad_input": to_pairs(x).sum(1).to(x.dtype)}
    weight = s["weight"].float()
    if case["direction"] == "forward":
        return {"out": (to_pairs(x) * weight.unsqueeze(-1)).sum(1).to(x.dtype)}
    grad = s["grad"].float().unsqueeze(1)
    return {"grad_rows": to_rows(grad * weight.unsqueeze(-1)), "grad_weights": (to_pairs(x) * grad).sum(-1).to(s["weight"].dtype)}


def _plain_quant(s):
    x = s["x"]
    out = {"values": _values(*_quantise(x))[:, : x.shape[1]].to(x.dtype)}
    if s["case"]["transposed"]:
        out["values_t"] = _values(*_quantise(x.t()))[:, : x.shape[0]].to(x.dtype)
    return out


def _plain_product(s):
    case, out = s["case"], DTYPES[s["case"]["out"]]
    a, w = _values(*_quantise(s["x"])), _unpack(s["w"], s["w_scale"])
    if not case["experts"]:
        return {"out": (a @ w.t()).to(out)}
    if case["gathered"]:
        a = a[s["gather"].long()]
    y = torch.cat([rows @ we.t() for rows, we in zip(a.split(s["splits_host"]), w)])
    if case["weighted"]:
        y = y * s["row_weight"].unsqueeze(-1)
    return {"rows": y.to(out)}


# ---- the framework's operators -----------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _flux():
    import flux_amd

    return flux_amd


@functools.lru_cache(maxsize=None)
def _quantiser(dtype):
    return _flux().Quantization(DTYPES[dtype], torch.float4_e2m1fn_x2)


@functools.lru_cache(maxsize=None)
def _gemm(out):
    return _flux().MxGemm(DTYPES[out])


def _own_moe(s):
    case, flux = s["case"], _flux()
    if case["kind"] == "permute":
        if case["direction"] == "forward":
            return {"rows": flux.moe_permute(s["x"], s["scatter"])}
        return {"grad_input": flux.moe_permute_backward(s["x"], s["scatter"])}
    if case["direction"] == "forward":
        return {"out": flux.moe_unpermute(s["x"], s["scatter"], s["weight"])}
    grad_rows, grad_weights = flux.moe_unpermute_backward(s["grad"], s["x"], s["scatter"], s["weight"])
    return {"grad_rows": grad_rows, "grad_weights": grad_weights}


def _own_quant(s):
    x, quant, transposed = s["x"], _quantiser(s["case"]["dtype"]), s["case"]["transposed"]
    codes, scale, codes_t, scale_t = quant.quantize_mx(x, return_tranpose=transposed)
    out = {"values": quant.dequantize_mx(codes, scale, x.shape[1])}
    if transposed:
        out["values_t"] = quant.dequantize_mx(codes_t, scale_t, x.shape[0])
    return out


def _own_product(s):
    case = s["case"]
    gemm = _gemm(case["out"])
    codes, scale, _, _ = _quantiser(case["dtype"]).quantize_mx(s["x"])
    if not case["experts"]:
        return {"out": gemm.forward(codes, s["w"], scale, s["w_scale"])}
    return {"rows": gemm.forward_grouped(codes, s["splits"], s["w"], scale, s["w_scale"],
                                         gather_index=s["gather"] if case["gathered"] else None,
                                         row_scale=s["row_weight"] if case["weighted"] else None)}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"permute": _own_moe, "unpermute": _own_moe, "quant": _own_quant, "product": _own_product}[kind](state)
    return {"permute": _plain_moe, "unpermute": _plain_moe, "quant": _plain_quant, "product": _plain_product}[kind](state)


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------


def _exact_mx(x):
    """The values of x [rows, K] in MXFP4, in 64 bits: the exponent by logarithm, the code by its borders."""
    rows, k = x.shape
    x = torch.cat([x.double(), x.new_zeros(rows, -k % 32, dtype=torch.float64)], dim=1).view(rows, -1, 32)
    most = x.abs().amax(dim=2, keepdim=True)
    e = torch.floor(torch.log2(most))
    e = e - (torch.pow(2.0, e) > most).double() + (torch.pow(2.0, e + 1) <= most).double()
    scale = torch.pow(2.0, (e - 2).clamp(min=-127))
    scale = torch.where(most == 0, 1.0, scale)
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    a = x.abs() / scale
    low, high = torch.bucketize(a, border), torch.bucketize(a, border, right=True)
    code = torch.where(low % 2 == 0, low, high)  # the two differ on a border only
    value = torch.sign(x) * grid[code] * scale
    return torch.where(torch.isfinite(most), value, math.nan).view(rows, -1)


def _exact_codes(codes, scale):
    """The values of packed codes [rows, K / 2] with scales [rows, K / 32], in 64 bits."""
    codes, scale = codes.view(torch.uint8).long(), scale.view(torch.uint8).double()
    nibble = torch.stack([codes % 16, codes // 16], dim=2).view(codes.shape[0], -1)
    e, m = nibble % 8 // 2, (nibble % 2).double()
    value = torch.where(e == 0, 0.5 * m, torch.pow(2.0, e.double() - 1) * (1 + 0.5 * m))
    value = torch.where(nibble >= 8, -value, value)
    return value * torch.pow(2.0, scale - 127).repeat_interleave(32, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        out = {"values": _exact_mx(s["x"])[:, : case["cols"]]}
        if case["transposed"]:
            out["values_t"] = _exact_mx(s["x"].t())[:, : case["rows"]]
        return out
    if case["kind"] == "product":
        a = _exact_mx(s["x"])
        if not case["experts"]:
            return {"out": a @ _exact_codes(s["w"], s["w_scale"]).t()}
        y, at = [], 0
        for e, rows in enumerate(s["splits_host"]):
            mine = slice(at, at + rows)
            part = (a[s["gather"][mine].long()] if case["gathered"] else a[mine]) @ _exact_codes(s["w"][e], s["w_scale"][e]).t()
            y.append(part * s["row_weight"][mine, None].double() if case["weighted"] else part)
            at += rows
        return {"rows": torch.cat(y)}
    x, scatter, pairs = s["x"].double(), s["scatter"].long(), s["scatter"].numel()
    named = scatter >= 0
    token = torch.arange(case["tokens"], device=x.device).unsqueeze(1).expand_as(scatter)
    if case["kind"] == "permute" and case["direction"] == "forward":
        rows = x.new_zeros(pairs, case["hidden"])
        rows[scatter[named]] = x[token[named]]
        return {"rows": rows}
    total = x.new_zeros(case["tokens"], case["hidden"])
    if case["kind"] == "permute":
        return {"grad_input": total.index_add_(0, token[named], x[scatter[named]])}
    w = s["weight"].double()
    if case["direction"] == "forward":
        return {"out": total.index_add_(0, token[named], x[scatter[named]] * w[named].unsqueeze(1))}
    grad = s["grad"].double()
    grad_rows, grad_weights = x.new_zeros(pairs, case["hidden"]), torch.zeros_like(w)
    grad_rows[scatter[named]] = grad[token[named]] * w[named].unsqueeze(1)
    grad_weights[named] = (grad[token[named]] * x[scatter[named]]).sum(1)
    return {"grad_rows": grad_rows, "grad_weights": grad_weights}


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _experts_hit(case):
    """Expected number of experts with at least one row."""
    t, k, e = case["tokens"], case["topk"], case["experts"]
    if not e:
        return 1
    if case["routing"] == "zipf":
        p = [(i + 1) ** -1.2 for i in range(e)]
        share = [min(1.0, k * v / sum(p)) for v in p]
    else:
        share = [k / e] * e
    return sum(1.0 - (1.0 - s) ** t for s in share)


def work(case):
    """Inputs read once, outputs written once, the weights of the experts that are hit read once."""
    size = {"bf16": 2, "f16": 2, "f32": 4}
    item = size[case["dtype"]]
    if case["kind"] == "quant":
        n, ways = case["rows"] * case["cols"], 2 if case["transposed"] else 1
        return {"bytes": n * item * (1 + ways) + ways * n * 17 // 32, "flops": 0}
    t, k, h = case["tokens"], case["topk"], case["hidden"]
    m = t * k if case.get("experts") else t
    if case["kind"] == "product":
        f, kb = case["ffn"], -(-h // BLOCK)
        rows = m if case["experts"] and not case["gathered"] else t
        weights = _experts_hit(case) * f * kb * 17
        return {"bytes": int(weights) + rows * h * item + m * f * size[case["out"]] + m * 8, "flops": 2 * m * h * f}
    routed = round(m * (1 - case["dropped"]))
    one = t * h * item + routed * h * item + m * 4
    if case["kind"] == "permute":
        return {"bytes": one + ((m - routed) * h * item if case["direction"] == "forward" else 0), "flops": 0}
    if case["direction"] == "forward":
        return {"bytes": one + m * size[case["weights"]], "flops": 2 * routed * h}
    return {"bytes": one + m * h * item + 2 * m * size[case["weights"]], "flops": 3 * routed * h}


# ---- drawn cases ------------------------------------------------------------------------------------------------


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choices(["permute", "unpermute", "quant", "product"], [3, 4, 3, 5])[0]
    if kind == "quant":
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": _log_int(rng, 1, 16384),
                "cols": _log_int(rng, 32, 16384), "transposed": rng.random() < 0.5}
    topk = rng.choice([1, 2, 2, 3, 4, 6, 8])
    case = {"kind": kind, "tokens": _log_int(rng, 1, 16384), "topk": topk, "experts": _log_int(rng, max(4, topk), 96),
            "routing": rng.choice(["softmax", "uniform", "zipf"])}
    if kind == "product":
        case.update(dtype=rng.choice(["bf16", "f16"]), out=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    hidden=128 * rng.randint(4, 112), ffn=128 * _log_int(rng, 4, 112), gathered=rng.random() < 0.5,
                    weighted=rng.random() < 0.4)
        if rng.random() < 0.4:  # widths that are not whole tiles or blocks
            case["hidden"] -= rng.randint(1, 127)
            case["ffn"] -= rng.randint(1, 127)
        if rng.random() < 0.15:
            case.update(experts=0, topk=1, gathered=False, weighted=False)
        return case
    case.update(direction=rng.choice(["forward", "backward"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                hidden=64 * _log_int(rng, 2, 128), dropped=rng.choice([0.0, 0.0, 0.0, 0.02, 0.1, 0.5]))
    if rng.random() < 0.3:
        case["hidden"] -= rng.randint(1, 63)
    if kind == "unpermute":
        case["weights"] = rng.choice(["f32", "f32", case["dtype"]])
    return case


def draw(rng):
    """One more case of the same ranges: no more bytes or arithmetic than the largest listed one, weights and rows that fit many times."""
    largest = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in largest), max(w["flops"] for w in largest)
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] <= bytes_ and w["flops"] <= flops and max(case.get("experts", 1), 1) * case.get("ffn", 0) * case.get("hidden", 0) <= 6e8:
            return case
