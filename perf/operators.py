"""The token operators around the recurrent core: the cases they are measured at, and their plain forms.

* ``lookup`` / ``gradient``: token ids to drive rows, ``scale * table[token]``, and the table's gradient
  (ids outside the table stand for "no stimulus": a zero row that takes no gradient);
* ``quantize``: a dense matrix into NVFP4 (E2M1 codes, an E4M3 scale per 16 elements of a row, a float32
  scale per row or for the whole matrix), also of the transpose, and read back;
* ``readout`` / ``train``: states times packed weights (``y = Q(x) W^T + b``), and a training step
  (``y``, and with operands quantised along each product's own axis ``dx``, ``dW`` and ``db``);
* ``logits``: penalties for repeated tokens, biases and grammar masks on logits, and the greedy choice.

A packed matrix of R rows and K columns is held as ``codes`` [R, 16 * ceil(K / 32)] (two codes per byte, the
even column in the low nibble), ``block_scales`` [ceil(R / 128), 4 * ceil(K / 256), 512] (E4M3 bytes: tile (i, j)
holds rows 128 i .. and blocks 4 j .., the scale of row r and block b at byte 16 (r % 32) + 4 (r % 128 // 32) + b % 4)
and ``scale`` [R] or [1]; everything beyond R and K is zero.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_PRODUCT = 8192 * 8192 * 4096  # multiply-adds of the largest product
MOST_VALUES = 64 << 20             # values of the largest lookup, table, matrix or logits
MOST_BYTES = 512 << 20             # what the largest drawn case reads and writes


def listed():
    return [
        # One tick of one network of 4,096 neurons (the framework's small graph): a call that is all latency.
        {"name": "lookup_tick", "op": "lookup", "tokens": 1, "neurons": 4096, "table": 32000, "dtype": "f32", "wide": False},
        # Drive for a streamed window of 20 ticks of the 166k-neuron graph at B = 8, float32 from a bf16 table.
        {"name": "lookup_window", "op": "lookup", "tokens": 160, "neurons": 166000, "table": 257, "dtype": "bf16", "wide": True},
        # The table's gradient after a short training window; odd token count, a 1,024-neuron core.
        {"name": "gradient_window", "op": "gradient", "tokens": 1999, "neurons": 1024, "table": 32000, "dtype": "f32"},
        # ... and after a large batch of sequences, with a few tokens that make up most of it.
        {"name": "gradient_batch", "op": "gradient", "tokens": 32768, "neurons": 2048, "table": 16384, "dtype": "bf16"},
        # A handful of states into NVFP4 before a readout: 8 networks of 50,000 neurons.
        {"name": "quantize_states", "op": "quantize", "rows": 8, "columns": 50000, "dtype": "f32", "per": "row", "transpose": False},
        # The transposed operand of a weight gradient, one scale for the matrix; neither side a multiple of a tile.
        {"name": "quantize_transposed", "op": "quantize", "rows": 8190, "columns": 4104, "dtype": "bf16", "per": "tensor", "transpose": True},
        # The next token of one network: one state against a vocabulary.
        {"name": "readout_token", "op": "readout", "rows": 1, "columns": 4096, "outputs": 32000, "dtype": "f32"},
        # Eight 50,000-neuron networks read out to an odd number of classes: a long sum and few outputs.
        {"name": "readout_wide", "op": "readout", "rows": 8, "columns": 50000, "outputs": 1001, "dtype": "f32"},
        # All states of a recorded window read out at once.
        {"name": "readout_window", "op": "readout", "rows": 4096, "columns": 4096, "outputs": 16384, "dtype": "bf16"},
        # One training step of the readout on a batch of states: the largest call.
        {"name": "train_batch", "op": "train", "rows": 8192, "columns": 4096, "outputs": 8192, "dtype": "bf16"},
        # The logits of one network with a short history.
        {"name": "logits_token", "op": "logits", "rows": 1, "vocabulary": 32000, "history": 17, "dtype": "f32"},
        # A full batch over a large vocabulary with long ragged histories.
        {"name": "logits_batch", "op": "logits", "rows": 256, "vocabulary": 131071, "history": 4096, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    case = _draw(rng)
    while work(case)["bytes"] > MOST_BYTES:
        case["tokens" if "tokens" in case else "rows"] //= 2
    return case


def _draw(rng):
    op = rng.choice(["lookup", "gradient", "quantize", "readout", "readout", "train", "logits"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "lookup":
        neurons = _spread(rng, 64, 166000)
        return {"op": op, "tokens": _spread(rng, 1, max(1, min(32768, MOST_VALUES // 2 // neurons))), "neurons": neurons,
                "table": _spread(rng, 2, max(2, min(131072, MOST_VALUES // neurons))), "dtype": dtype, "wide": rng.random() < 0.5}
    if op == "gradient":
        neurons = _spread(rng, 64, 16384)
        return {"op": op, "tokens": _spread(rng, 1, min(65536, MOST_VALUES // neurons)), "neurons": neurons,
                "table": _spread(rng, 2, min(131072, MOST_VALUES // neurons)), "dtype": dtype}
    if op == "quantize":
        columns = _spread(rng, 16, 50000)
        return {"op": op, "rows": _spread(rng, 1, min(16384, MOST_VALUES // 2 // columns)), "columns": columns, "dtype": dtype,
                "per": rng.choice(["row", "tensor"]), "transpose": rng.random() < 0.5}
    if op == "readout":
        columns, rows = _spread(rng, 64, 50000), _spread(rng, 1, 8192)
        rows = min(rows, MOST_VALUES // columns)
        return {"op": op, "rows": rows, "columns": columns, "dtype": dtype,
                "outputs": _spread(rng, 2, max(2, min(131072, 2 * MOST_VALUES // columns, 2 * MOST_VALUES // rows, MOST_PRODUCT // (rows * columns))))}
    if op == "train":
        columns, rows = _spread(rng, 64, 8192), _spread(rng, 16, 8192)
        return {"op": op, "rows": rows, "columns": columns, "outputs": _spread(rng, 16, min(16384, MOST_PRODUCT // (rows * columns))), "dtype": dtype}
    vocabulary = _spread(rng, 64, 262144)
    return {"op": op, "rows": _spread(rng, 1, max(1, min(512, MOST_VALUES // 2 // vocabulary))), "vocabulary": vocabulary,
            "history": rng.choice([0, _spread(rng, 1, 16384)]), "dtype": dtype}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _ids(count, table, g):
    """Token ids as they occur: a few are frequent (log-uniform ranks), one in 32 is -1, no stimulus."""
    u = torch.rand(count, generator=g, device="cuda")
    ids = (torch.exp(u * math.log(table + 1.0)) - 1.0).to(torch.int64).clamp_(0, table - 1)
    return torch.where(torch.rand(count, generator=g, device="cuda") < 1 / 32, -1, ids)


def _states(rows, columns, dtype, g):
    """Soma states: in [0, 1], about a third of them silent."""
    return (torch.rand(rows, columns, generator=g, device="cuda") * 1.5 - 0.5).clamp_(0.0, 1.0).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype = case["op"], TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std)

    s = {"case": case}
    if op == "lookup":
        s["table"] = normal(case["table"], case["neurons"], std=0.02).to(dtype)
        s["tokens"] = _ids(case["tokens"], case["table"], g)
        s["scale"] = math.sqrt(case["neurons"])
    elif op == "gradient":
        s["grad"] = normal(case["tokens"], case["neurons"], std=1e-3).to(dtype)
        s["tokens"] = _ids(case["tokens"], case["table"], g)
        s["scale"] = math.sqrt(case["neurons"])
    elif op == "quantize":
        s["value"] = normal(case["rows"], case["columns"]).to(dtype)
    elif op == "readout":
        s["state"] = _states(case["rows"], case["columns"], dtype, g)
        s["weight"] = _pack(normal(case["outputs"], case["columns"], std=case["columns"] ** -0.5), "tensor")
        s["bias"] = normal(case["outputs"], std=0.1)
    elif op == "train":
        s["state"] = _states(case["rows"], case["columns"], dtype, g).requires_grad_()
        s["weight"] = normal(case["outputs"], case["columns"], std=case["columns"] ** -0.5).to(dtype).requires_grad_()
        s["bias"] = normal(case["outputs"], std=0.1).requires_grad_()
        s["grad"] = normal(case["rows"], case["outputs"], std=0.1).to(dtype)
    else:
        rows, vocabulary, history = case["rows"], case["vocabulary"], case["history"]
        s["logits"] = normal(rows, vocabulary, std=3.0).to(dtype)
        s["history"] = _ids(rows * history, vocabulary, g).view(rows, history).to(torch.int32)
        s["lengths"] = torch.randint(0, history + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["prompt_lengths"] = (s["lengths"] * torch.rand(rows, generator=g, device="cuda")).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["bias"] = normal(vocabulary, std=0.5)
        # About half of each row's tokens are allowed; the last row of a batch has nothing left.
        s["mask"] = torch.randint(-(1 << 31), 1 << 31, (rows, (vocabulary + 31) // 32), generator=g, device="cuda").to(torch.int32)
        if rows > 1:
            s["mask"][-1] = 0
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _tensor_scale(value):
    amax = value.detach().abs().amax().reshape(1).float()
    return (amax / torch.full_like(amax, 2688.0)).clamp_min(torch.finfo(torch.float32).tiny)


def _quantize(value, per, scale=None):
    """(codes 0..15 [R, blocks, 16], E4M3 block scales [R, blocks], float32 scale [R] or [1]) of a matrix."""
    value = value.detach().float()
    blocks = torch.nn.functional.pad(value, (0, -value.shape[1] % 16)).view(value.shape[0], -1, 16)
    size = blocks.abs()
    most = size.amax(-1)
    if scale is None and per == "row":
        amax = most.amax(-1)
        scale = (amax / torch.full_like(amax, 2688.0)).clamp_min(torch.finfo(torch.float32).tiny)
    elif scale is None:
        scale = _tensor_scale(value)
    block = (most / (6.0 * scale).unsqueeze(-1)).clamp_max(448.0).to(torch.float8_e4m3fn)
    step = scale.unsqueeze(-1) * block.float()
    size = size / torch.where(step > 0, step, 1.0).unsqueeze(-1)
    code = torch.zeros_like(size, dtype=torch.uint8)
    for i, middle in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # a tie goes to the even code
        code += (size >= middle) if i % 2 else (size > middle)
    return code | (blocks.signbit().to(torch.uint8) << 3), block, scale


def _values(code, block, scale, columns, dtype=torch.float32):
    """The values that a quantised matrix stands for [R, columns]."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device, dtype=dtype)
    levels = torch.cat([levels, -levels])
    step = block.to(dtype) * scale.to(dtype).unsqueeze(-1)
    return (levels[code.int()] * step.unsqueeze(-1)).flatten(1)[:, :columns]


def _quantized(value, per):
    return _values(*_quantize(value, per), value.shape[1])


def _pack(value, per):
    """The packed matrix of `value`, some rows at a time where it is large."""
    rows, columns = value.shape
    scale = None if per == "row" else _tensor_scale(value)
    code, block, scales = [], [], []
    for part in value.split(max(1, (32 << 20) // columns)):
        c, b, s = _quantize(part, per, scale)
        c = torch.nn.functional.pad(c.flatten(1), (0, -c[0].numel() % 32))
        code.append(c[:, 0::2] | (c[:, 1::2] << 4))
        block.append(b.view(torch.uint8))
        scales.append(s)
    block = torch.cat(block)
    block = torch.nn.functional.pad(block, (0, -block.shape[1] % 16, 0, -rows % 128))
    tiles = block.view(-1, 4, 32, block.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, block.shape[1] // 4, 512)
    return {"codes": torch.cat(code), "block_scales": tiles.contiguous(), "scale": torch.cat(scales) if scale is None else scale, "columns": columns}


def _unpack(packed, dtype=torch.float32):
    """The values of a packed matrix."""
    codes, tiles, columns = packed["codes"], packed["block_scales"], packed["columns"]
    blocks = (columns + 15) // 16
    block = tiles.view(*tiles.shape[:2], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    block = block[: codes.shape[0], :blocks].contiguous().view(torch.float8_e4m3fn)
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, : 16 * blocks].reshape(codes.shape[0], blocks, 16)
    return _values(code, block, packed["scale"], columns, dtype)


def _counts(s):
    """(occurrences among the generated tokens [B, V], whether the token occurs at all [B, V])."""
    rows, vocabulary = s["logits"].shape
    history = s["history"].long()
    at = torch.arange(history.shape[1], device=history.device)
    valid = (at < s["lengths"].unsqueeze(1)) & (history >= 0) & (history < vocabulary)
    generated = valid & (at >= s["prompt_lengths"].unsqueeze(1))
    index = history.clamp(0, vocabulary - 1)
    count = torch.zeros(rows, vocabulary, device=history.device, dtype=torch.int32).scatter_add_(1, index, generated.int())
    seen = torch.zeros(rows, vocabulary, device=history.device, dtype=torch.int32).scatter_add_(1, index, valid.int())
    return count, seen > 0


def _allowed(s):
    vocabulary = s["logits"].shape[1]
    bits = torch.arange(32, device="cuda", dtype=torch.int32)
    return ((s["mask"].unsqueeze(-1) >> bits) & 1).flatten(1)[:, :vocabulary] != 0


def _choice(logits):
    """The lowest index of a row's largest value, -1 where nothing is above -inf."""
    most = logits.amax(1, keepdim=True)
    at = torch.arange(logits.shape[1], device=logits.device)
    first = torch.where(logits == most, at, logits.shape[1]).amin(1)
    return torch.where(most.squeeze(1) > -math.inf, first, -1)


def run(s):
    return _own(s) if own else _plain(s)


def _plain(s):
    case, dtype = s["case"], TYPES[s["case"]["dtype"]]
    op = case["op"]
    if op == "lookup":
        table, tokens = s["table"], s["tokens"]
        rows = table[tokens.clamp(0, table.shape[0] - 1)].float() * s["scale"]
        valid = (tokens >= 0) & (tokens < table.shape[0])
        return torch.where(valid.unsqueeze(1), rows, 0.0).to(torch.float32 if case["wide"] else dtype)
    if op == "gradient":
        valid = (s["tokens"] >= 0) & (s["tokens"] < case["table"])
        total = torch.zeros(case["table"], case["neurons"], device="cuda")
        total.index_add_(0, torch.where(valid, s["tokens"], 0), torch.where(valid.unsqueeze(1), s["grad"].float(), 0.0))
        return (total * s["scale"]).to(dtype)
    if op == "quantize":
        value = s["value"].t() if case["transpose"] else s["value"]
        code, block, scale = _quantize(value, case["per"])
        return {"values": _values(code, block, scale, value.shape[1]).to(dtype), "scale": scale}
    if op == "readout":
        return (_quantized(s["state"], "row") @ _unpack(s["weight"]).t() + s["bias"]).to(dtype)
    if op == "train":
        x, w, d = s["state"].detach(), s["weight"].detach(), s["grad"]
        y = _quantized(x, "row") @ _quantized(w, "tensor").t() + s["bias"].detach()
        dx = _quantized(d, "row") @ _quantized(w.t(), "tensor").t()
        dw = _quantized(d.t(), "tensor") @ _quantized(x.t(), "tensor").t()
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype), "db": d.float().sum(0)}
    count, seen = _counts(s)
    x = s["logits"].float()
    r = s["repetition"].unsqueeze(1)
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"].unsqueeze(1) * count
    x = x - torch.where(count > 0, s["presence"].unsqueeze(1), 0.0)
    x = torch.where(_allowed(s), x + s["bias"], -math.inf).to(dtype)
    return {"logits": x, "choice": _choice(x)}


def _own(s):
    import neurosim_gpu_b200 as nsb

    case, dtype = s["case"], TYPES[s["case"]["dtype"]]
    op = case["op"]
    if op == "lookup":
        return nsb.stimulus_drive(s["tokens"], s["table"], scale=s["scale"], dtype=torch.float32 if case["wide"] else dtype)
    if op == "gradient":
        return nsb.stimulus_gradient(s["tokens"], s["grad"], case["table"], scale=s["scale"])
    if op == "quantize":
        packed = nsb.quantize_nvfp4(s["value"], per=case["per"], transpose=case["transpose"])
        return {"values": packed.dequantize(dtype), "scale": packed.scale}
    if op == "readout":
        w = s["weight"]
        weight = nsb.Nvfp4Matrix(w["codes"], w["block_scales"], w["scale"], w["columns"])
        return nsb.nvfp4_readout(s["state"], weight, s["bias"])
    if op == "train":
        y = nsb.nvfp4_readout(s["state"], s["weight"], s["bias"])
        dx, dw, db = torch.autograd.grad(y, (s["state"], s["weight"], s["bias"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    logits, choice = nsb.adjust_logits(
        s["logits"], history=s["history"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias=s["bias"], mask=s["mask"], choose=True)
    return {"logits": logits, "choice": choice}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _packed_bytes(rows, columns):
    return rows * (columns / 2 + (columns + 15) // 16)


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "lookup":
        touched = min(case["tokens"], case["table"])
        return {"bytes": touched * case["neurons"] * e + 8 * case["tokens"] + case["tokens"] * case["neurons"] * (4 if case["wide"] else e),
                "flops": case["tokens"] * case["neurons"]}
    if op == "gradient":
        return {"bytes": (case["tokens"] + case["table"]) * case["neurons"] * e + 8 * case["tokens"], "flops": case["tokens"] * case["neurons"]}
    if op == "quantize":
        return {"bytes": 2 * case["rows"] * case["columns"] * e + 2 * _packed_bytes(case["rows"], case["columns"]),
                "flops": 4 * case["rows"] * case["columns"]}
    if op == "readout":
        m, k, n = case["rows"], case["columns"], case["outputs"]
        return {"bytes": m * k * e + _packed_bytes(n, k) + 4 * n + m * n * e, "flops": 2 * m * k * n}
    if op == "train":
        m, k, n = case["rows"], case["columns"], case["outputs"]
        return {"bytes": 2 * (m * k + n * k + m * n) * e + 8 * n, "flops": 6 * m * k * n}
    b, v = case["rows"], case["vocabulary"]
    return {"bytes": 2 * b * v * e + b * (4 * ((v + 31) // 32) + 4 * case["history"] // 2 + 28) + 4 * v, "flops": 5 * b * v}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------


def _nvfp4_exact(value, per):
    """The float64 values that NVFP4 gives a matrix, from the format's definition: the scale is a float32, a block's
    scale an E4M3 number, and a code the nearest level to the float32 quotient |x| / (scale * block scale)."""
    v = value.detach().to(torch.float64)
    rows, columns = v.shape
    whole = torch.zeros(rows, (columns + 15) // 16 * 16, dtype=torch.float64, device=v.device)
    whole[:, :columns] = v
    whole = whole.reshape(rows, -1, 16)
    top = whole.abs().amax((1, 2), keepdim=True) if per == "row" else whole.abs().amax().reshape(1, 1, 1)
    scale = (top / 2688.0).to(torch.float32).clamp(min=2.0 ** -126)
    bound = whole.abs().amax(2, keepdim=True).to(torch.float32) / (scale * 6.0)
    block = torch.minimum(bound, torch.full_like(bound, 448.0)).to(torch.float8_e4m3fn).to(torch.float32)
    unit = scale * block
    unit = torch.where(unit > 0, unit, torch.ones_like(unit))
    ratio = (whole.abs().to(torch.float32) / unit).to(torch.float64)
    # Levels are 0.5 apart up to 2, 1 apart up to 4, then 2 apart; torch.round takes ties to the even multiple.
    near = torch.where(ratio < 2.0, torch.round(ratio * 2.0) / 2.0, torch.where(ratio < 4.0, torch.round(ratio), torch.round(ratio / 2.0) * 2.0))
    near = near.clamp(max=6.0)
    return (torch.copysign(near, whole) * block.to(torch.float64) * scale.to(torch.float64)).reshape(rows, -1)[:, :columns], scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        padded = torch.cat([s["table"].double() * s["scale"], torch.zeros(1, case["neurons"], dtype=torch.float64, device="cuda")])
        inside = (s["tokens"] >= 0) & (s["tokens"] < case["table"])
        return padded[torch.where(inside, s["tokens"], case["table"])]
    if op == "gradient":
        order = torch.where((s["tokens"] < 0) | (s["tokens"] >= case["table"]), case["table"], s["tokens"])
        total = torch.zeros(case["table"] + 1, case["neurons"], dtype=torch.float64, device="cuda")
        return total.index_add(0, order, s["grad"].double())[:-1] * s["scale"]
    if op == "quantize":
        value, scale = _nvfp4_exact(s["value"].t() if case["transpose"] else s["value"], case["per"])
        return {"values": value, "scale": scale.reshape(-1).double()}
    if op == "readout":
        weight = torch.cat([_unpack({**s["weight"], "codes": c, "block_scales": t}, torch.float64) for c, t in
                            zip(s["weight"]["codes"].split(8192), s["weight"]["block_scales"].split(64))])
        return _nvfp4_exact(s["state"], "row")[0] @ weight.t() + s["bias"].double()
    if op == "train":
        x, w, d = s["state"].detach(), s["weight"].detach(), s["grad"]
        return {"y": _nvfp4_exact(x, "row")[0] @ _nvfp4_exact(w, "tensor")[0].t() + s["bias"].detach().double(),
                "dx": _nvfp4_exact(d, "row")[0] @ _nvfp4_exact(w.t(), "tensor")[0].t(),
                "dw": _nvfp4_exact(d.t(), "tensor")[0] @ _nvfp4_exact(x.t(), "tensor")[0].t(),
                "db": d.double().sum(0)}
    count, seen = _counts(s)
    x, r = s["logits"].double(), s["repetition"].double().unsqueeze(1)
    x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x))
    x = x - count * s["frequency"].double().unsqueeze(1) - (count > 0) * s["presence"].double().unsqueeze(1) + s["bias"].double()
    return {"logits": x.masked_fill(~_allowed(s), -math.inf), "choice": None}
