"""Timed cases of the 8-bit linear layers of a DiT block, with their plain forms.

Values are held as e4m3 with one power of two (e8m0) for each group of 128 along a
row of activations, or for each block of 128 x 128 of a weight: the smallest power
of two by which no value of the group passes 448, e4m3's largest. Every case is one
pass through one operator:

* ``quantize`` - ``quantize_fp8``: rows of activations, and ``quantize_fp8_weight``:
  a weight's blocks;
* ``norm``     - ``fused_rmsnorm_modulate_fp8`` and
  ``fused_residual_gate_rmsnorm_modulate_fp8``: the norms and modulation before a
  linear layer, their result in 8 bits;
* ``linear``   - ``fused_linear_fp8``: the matrix product of 8-bit operands (or of
  bf16 rows, which it rounds to 8 bits first) with bias, activation or gated
  activation, gate and residual behind it, its result in bf16 or in 8 bits for the
  layer after it.

The framework is inference only, so there is no backward direction.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
GROUP = 128  # values that share a scale
LARGEST = 448.0  # of e4m3
TABLE_ROWS = 9  # modulation rows of a block
MAX_FLOPS = 2 * 6240 * 5376 * 28672  # the largest listed cases
MAX_VALUES = 28672 * 5376


def listed() -> list[dict]:
    return [
        # The timestep rows of a block before their projection: latency.
        _quantize("quantize_9", 9, 5376),
        # The attention's output on one Ulysses rank (480p / 5 s, 40 heads), before the output projection.
        _quantize("quantize_rank", 6240, 5120),
        # A gated up weight when a model is loaded, or its layer is swapped in.
        _quantize("quantize_weight_up", 28672, 5376, "gated"),
        # The norm before a branch at the microbenchmark's row count: latency.
        _norm("norm8_257", "modulate", 257, 5376, "bf16"),
        # The norm between the attention and the MLP on one rank's rows.
        _norm("norm8_rank", "residual", 6240, 5376, "bf16"),
        # The projection of one timestep's embedding: a single token.
        _linear("linear8_1_token", 1, 1024, 1024, "bf16", activation="silu", bias="bf16"),
        # The modulation rows of a block: bound by reading the weights.
        _linear("linear8_modulation_rows", 9, 5376, 6 * 5376, "bf16", bias="bf16"),
        # The audio segment's 1,296 tokens and one more through an odd-width adapter with a GELU, back onto the residual.
        _linear("linear8_ragged_gelu", 1297, 1552, 2056, "fp8", activation="gelu_tanh", bias="f32", residual=True),
        # One latent frame's tokens on one of four ranks: fewer tiles than the card has units.
        _linear("linear8_frame_rank", 390, 5376, 5376, "bf16", residual=True, gate="f32"),
        # MLP up of one Ulysses rank at 480p / 5 s: the gated activation, its result in 8 bits for the layer below.
        _linear("mlp8_up_rank", 6240, 5376, 14336, "fp8", activation="silu", gated=True, out="fp8"),
        # MLP down of the same rows, with the gated residual of the block.
        _linear("mlp8_down_rank", 6240, 14336, 5376, "fp8", bias="bf16", residual=True, gate="bf16"),
        # The q/k/v projection of the same rows from bf16 activations.
        _linear("linear8_qkv_rank", 6240, 5120, 15360, "bf16", bias="bf16"),
    ]


def _quantize(name, rows, cols, weight="no", dtype="bf16"):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "weight": weight, "dtype": dtype}


def _norm(name, kind, rows, cols, tables, weights="bf16"):
    return {"name": name, "op": "norm", "kind": kind, "rows": rows, "cols": cols, "tables": tables, "weights": weights}


def _linear(name, m, k, n, x, activation="none", gated=False, bias="none", residual=False, gate="none", out="bf16"):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "x": x, "activation": activation, "gated": gated, "bias": bias,
            "residual": residual, "gate": gate, "out": out}


def draw(rng) -> dict:
    """One more case: the same operators, sizes spread over their ranges."""

    def log_int(lo: int, hi: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["linear", "linear", "linear", "linear", "norm", "norm", "quantize", "quantize"])
    if op == "linear":
        m = log_int(1, 64) if rng.random() < 0.35 else log_int(64, 12480)
        k, n = 16 * log_int(4, 896), 16 * log_int(4, 896)
        gated = rng.random() < 0.3
        while 2 * m * k * n * (1 + gated) > MAX_FLOPS:
            m = m // 2
        out = "fp8" if rng.random() < 0.3 else "bf16"
        residual = not gated and out == "bf16" and rng.random() < 0.5
        case = _linear("", m, k, n, rng.choice(["bf16", "fp8", "fp8"]), rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                       gated, rng.choice(["none", "bf16", "f32"]), residual, rng.choice(["none", "bf16", "f32"]) if residual else "none", out)
    elif op == "norm":
        cols = rng.choice([1024, 2064, 5120, 5376, 6144, 1008]) if rng.random() < 0.6 else 16 * log_int(4, 512)
        case = _norm("", rng.choice(["modulate", "residual"]), log_int(1, 12480), cols, rng.choice(["bf16", "bf16", "f32"]),
                     rng.choice(["bf16", "f32"]))
    else:
        rows, cols = log_int(1, 28672), 16 * log_int(4, 896)
        while rows * cols > MAX_VALUES // 2:
            rows = rows // 2
        weight = rng.choice(["no", "no", "plain", "gated"])
        case = _quantize("", 2 * rows if weight == "gated" else rows, cols, weight, rng.choice(["bf16", "bf16", "f32"]))
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed: int) -> None:
        self.device = torch.device("cuda:0")
        self.generator = torch.Generator(device=self.device).manual_seed(seed)

    def normal(self, *shape: int, dtype: torch.dtype = torch.bfloat16, scale: float = 1.0) -> torch.Tensor:
        return torch.randn(shape, device=self.device, generator=self.generator).mul_(scale).to(dtype)

    def activations(self, rows: int, cols: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """Rows whose channels differ in size, as activations do."""
        channel = torch.randn((cols,), device=self.device, generator=self.generator).mul_(0.7).exp_()
        return torch.randn((rows, cols), device=self.device, generator=self.generator).mul_(channel).to(dtype)

    def gain(self, n: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return (1.0 + self.normal(n, dtype=torch.float32, scale=0.1)).to(dtype)

    def index(self, rows: int) -> torch.Tensor:
        """The modulation row of each token: frames in order."""
        return torch.arange(rows, device=self.device) * TABLE_ROWS // max(rows, 1)


_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _held(q: torch.Tensor, scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Values and scales as the framework's quantisation hands them on: rows of
    scales start at multiples of 16 bytes."""
    r, c = scale.shape
    rows = scale.new_zeros((r, c + -c % 16), dtype=torch.uint8)
    rows[:, :c] = scale.view(torch.uint8)
    return q, rows[:, :c].view(torch.float8_e8m0fnu)


def prepare(case: dict, seed: int) -> dict:
    rng = _Inputs(seed)
    op = case["op"]
    s: dict = {"op": op}
    if op == "quantize":
        s["weight"] = case["weight"]
        dtype = _DTYPES[case["dtype"]]
        if case["weight"] == "no":
            s["x"] = rng.activations(case["rows"], case["cols"], dtype)
        else:
            s["x"] = rng.normal(case["rows"], case["cols"], dtype=dtype, scale=case["cols"] ** -0.5)
    elif op == "norm":
        rows, cols = case["rows"], case["cols"]
        s["kind"] = case["kind"]
        s["x"] = rng.activations(rows, cols)
        s["residual"] = rng.normal(rows, cols, scale=2.0) if case["kind"] == "residual" else None
        s["norm_weight"] = rng.gain(cols, _DTYPES[case["weights"]])
        tables = rng.normal(TABLE_ROWS, 3 * cols, dtype=_DTYPES[case["tables"]], scale=0.3)
        s["shift"], s["scale"], s["gate"] = tables.chunk(3, dim=-1)
        s["index"] = rng.index(rows)
    else:
        m, k, n = case["m"], case["k"], case["n"]
        rows = 2 * n if case["gated"] else n
        s["x"], s["x_scale"] = rng.activations(m, k), None
        if case["x"] == "fp8":
            s["x"], s["x_scale"] = _held(*_in_8_bits(s["x"]))
        weight = rng.normal(rows, k, scale=k**-0.5)
        s["weight"], s["weight_scale"] = _held(*_weight_in_8_bits(weight, case["gated"]))
        s["bias"] = None if case["bias"] == "none" else rng.normal(rows, dtype=_DTYPES[case["bias"]], scale=0.1)
        s["activation"] = None if case["activation"] == "none" else case["activation"]
        s["gated"] = case["gated"]
        s["quantize"] = case["out"] == "fp8"
        s["residual"] = rng.normal(m, n, scale=2.0) if case["residual"] else None
        s["gate"] = s["index"] = None
        if case["gate"] != "none":
            # one of the six modulation vectors that lie side by side in a row
            s["gate"] = rng.normal(TABLE_ROWS, 3 * n, dtype=_DTYPES[case["gate"]], scale=0.3).chunk(3, dim=-1)[2]
            s["index"] = rng.index(m)
    return s


# ---------------------------------------------------------------- plain forms, 32 bits


def _exponent(top: torch.Tensor) -> torch.Tensor:
    """e8m0's byte of groups whose largest magnitude is ``top``: of the smallest
    power of two s, 2^-126 at the least, with top <= 448 s; 255 (NaN) where top is
    not finite."""
    part, power = torch.frexp(top)  # top = part 2^power, 1/2 <= part < 1; 448 = 7/8 2^9
    byte = (power - 9 + (part > 0.875) + 127).clamp(1, 254)
    byte = torch.where(top < 2.0**-110, 1, byte)
    return torch.where(torch.isfinite(top), byte, 255).to(torch.uint8)


def _value(byte: torch.Tensor) -> torch.Tensor:
    value = torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127)
    return torch.where(byte == 255, float("nan"), value)


def _groups(x: torch.Tensor, rows: int) -> torch.Tensor:
    """(r, c) -> (groups of rows, rows, groups of columns, 128), filled up with zeros."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % GROUP, 0, -r % rows))
    return x.view(-1, rows, x.shape[1] // GROUP, GROUP)


def _in_8_bits(x: torch.Tensor, rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    r, c = x.shape
    x = _groups(x.float(), rows)
    byte = _exponent(x.abs().amax((1, 3)))
    q = x * (1.0 / _value(byte))[:, None, :, None]
    q = q.reshape(-1, x.shape[2] * GROUP)[:r, :c].to(torch.float8_e4m3fn)
    return q.contiguous(), byte.view(torch.float8_e8m0fnu)


def _weight_in_8_bits(w: torch.Tensor, gated: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Blocks of 128 x 128; of a gated weight those of the values, then those of the gates."""
    if not gated:
        return _in_8_bits(w, GROUP)
    (q0, s0), (q1, s1) = (_in_8_bits(half, GROUP) for half in w.chunk(2))
    return torch.cat((q0, q1)), torch.cat((s0.view(torch.uint8), s1.view(torch.uint8))).view(torch.float8_e8m0fnu)


def _values(q: torch.Tensor, scale: torch.Tensor, rows: int = 1) -> torch.Tensor:
    s = _value(scale.view(torch.uint8)).repeat_interleave(rows, 0)[: q.shape[0]]
    return q.float() * s.repeat_interleave(GROUP, 1)[:, : q.shape[1]]


def _weight_values(s: dict) -> torch.Tensor:
    if not s["gated"]:
        return _values(s["weight"], s["weight_scale"], GROUP)
    return torch.cat([_values(q, v, GROUP) for q, v in zip(s["weight"].chunk(2), s["weight_scale"].chunk(2))])


def _plain_quantize(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    return _in_8_bits(s["x"]) if s["weight"] == "no" else _weight_in_8_bits(s["x"], s["weight"] == "gated")


def _plain_norm(s: dict) -> tuple[torch.Tensor, ...]:
    t = s["index"]
    h = s["x"].float()
    if s["kind"] == "residual":
        h = s["residual"].float() + s["gate"].float()[t] * h
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["norm_weight"].float()
    y = _in_8_bits(y * (1.0 + s["scale"].float()[t]) + s["shift"].float()[t])
    return (h.to(torch.bfloat16), *y) if s["kind"] == "residual" else y


def _activate(z: torch.Tensor, kind: str | None) -> torch.Tensor:
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5**0.5))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z * (z > 0) if kind == "relu" else z


def _plain_linear(s: dict):
    x = _values(*(_in_8_bits(s["x"]) if s["x_scale"] is None else (s["x"], s["x_scale"])))
    z = x @ _weight_values(s).t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s["gated"]:
        value, act = z.chunk(2, dim=-1)
        y = value * _activate(act, s["activation"])
    else:
        y = _activate(z, s["activation"])
    if s["gate"] is not None:
        y = y * s["gate"].float()[s["index"]]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return _in_8_bits(y) if s["quantize"] else y.to(torch.bfloat16)


_PLAIN = {"quantize": _plain_quantize, "norm": _plain_norm, "linear": _plain_linear}


def _own(s: dict):
    op = s["op"]
    if op == "quantize":
        from h3_flash_amd import quantize_fp8, quantize_fp8_weight

        return quantize_fp8(s["x"]) if s["weight"] == "no" else quantize_fp8_weight(s["x"], gated=s["weight"] == "gated")
    if op == "norm":
        from h3_flash_amd.fusions import fused_residual_gate_rmsnorm_modulate_fp8, fused_rmsnorm_modulate_fp8

        rest = (s["norm_weight"], s["scale"], s["shift"], s["index"], EPS)
        if s["kind"] == "modulate":
            return fused_rmsnorm_modulate_fp8(s["x"], *rest)
        return fused_residual_gate_rmsnorm_modulate_fp8(s["residual"], s["x"], s["gate"], *rest)
    from h3_flash_amd import fused_linear_fp8

    return fused_linear_fp8(s["x"], s["weight"], s["weight_scale"], s["bias"], x_scale=s["x_scale"], activation=s["activation"],
                            gated=s["gated"], residual=s["residual"], gate=s["gate"], index=s["index"], quantize=s["quantize"])


def run(s: dict):
    return _own(s) if own else _PLAIN[s["op"]](s)


def work(case: dict) -> dict:
    size = {"none": 0, "fp8": 1, "bf16": 2, "f32": 4}
    up = lambda n: -(-n // GROUP)  # noqa: E731
    op = case["op"]
    if op == "quantize":
        n, c = case["rows"] * case["cols"], case["cols"]
        groups = case["rows"] if case["weight"] == "no" else up(case["rows"])
        return {"bytes": n * (size[case["dtype"]] + 1) + groups * up(c), "flops": 3 * n}
    if op == "norm":
        rows, c = case["rows"], case["cols"]
        tables = 3 if case["kind"] == "residual" else 2
        nbytes = rows * c * (7 if case["kind"] == "residual" else 3) + rows * (up(c) + 8)
        nbytes += c * (tables * TABLE_ROWS * size[case["tables"]] + size[case["weights"]])
        return {"bytes": nbytes, "flops": 12 * rows * c}
    m, k, n = case["m"], case["k"], case["n"]
    rows = 2 * n if case["gated"] else n
    nbytes = m * k * size[case["x"]] + rows * k + up(rows) * up(k) + m * n * (size[case["out"]] + (2 if case["residual"] else 0))
    nbytes += (m * up(k) if case["x"] == "fp8" else 0) + (m * up(n) if case["out"] == "fp8" else 0) + size[case["bias"]] * rows
    if case["gate"] != "none":
        nbytes += size[case["gate"]] * TABLE_ROWS * n + 8 * m
    return {"bytes": nbytes, "flops": 2 * m * k * rows}


# ---------------------------------------------------------------- 64 bits


def _round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """e4m3's nearest value, ties to even: steps of 2^(e - 3), 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def _exact_8_bits(y: torch.Tensor, rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    r, c = y.shape
    q = torch.empty_like(y)
    scale = torch.empty((-(-r // rows), -(-c // GROUP)), dtype=torch.float64, device=y.device)
    for j in range(scale.shape[1]):
        part = y[:, j * GROUP : (j + 1) * GROUP]
        if rows == 1:
            top = part.abs().amax(1)
        else:
            top = torch.stack([p.abs().max() for p in part.split(rows)])
        power = torch.ceil(torch.log2((top / LARGEST).clamp_min(2.0**-126)))
        # (log2 next to a whole number)
        power = torch.where(top <= LARGEST * torch.exp2(power - 1), power - 1, power)
        power = torch.where(top > LARGEST * torch.exp2(power), power + 1, power).clamp_min(-126)
        scale[:, j] = torch.exp2(power)
        q[:, j * GROUP : (j + 1) * GROUP] = _round_e4m3(part / scale[:, j].repeat_interleave(rows)[:r, None])
    return q, scale


def _exact_weight(w: torch.Tensor, gated: bool) -> tuple[torch.Tensor, torch.Tensor]:
    parts = [_exact_8_bits(half, GROUP) for half in w.chunk(2 if gated else 1)]
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_quantize(s: dict):
    x = s["x"].double()
    return _exact_8_bits(x) if s["weight"] == "no" else _exact_weight(x, s["weight"] == "gated")


def _exact_norm(s: dict):
    cols = (s["x"].shape[-1],)
    gate, scale, shift = (torch.index_select(s[n].double(), 0, s["index"]) for n in ("gate", "scale", "shift"))
    hidden = s["x"].double() if s["residual"] is None else torch.addcmul(s["residual"].double(), gate, s["x"].double())
    normed = torch.nn.functional.rms_norm(hidden, cols, s["norm_weight"].double(), EPS)
    out = _exact_8_bits(torch.addcmul(shift, normed, scale + 1.0))
    return out if s["residual"] is None else (hidden, *out)


def _exact_linear(s: dict):
    if s["x_scale"] is None:
        x, scale = _exact_8_bits(s["x"].double())
    else:
        x, scale = s["x"].double(), s["x_scale"].double()
    x = x * scale.repeat_interleave(GROUP, 1)[:, : x.shape[1]]
    halves = 2 if s["gated"] else 1
    z = []
    for w, v, b in zip(s["weight"].chunk(halves), s["weight_scale"].chunk(halves), (s["bias"].chunk(halves) if s["bias"] is not None else (None, None))):
        w = w.double() * v.double().repeat_interleave(GROUP, 0)[: w.shape[0]].repeat_interleave(GROUP, 1)[:, : w.shape[1]]
        z.append(torch.nn.functional.linear(x, w, None if b is None else b.double()))
    act = {
        None: lambda a: a,
        "silu": lambda a: a * torch.sigmoid(a),
        "gelu": lambda a: torch.nn.functional.gelu(a),
        "gelu_tanh": lambda a: torch.nn.functional.gelu(a, approximate="tanh"),
        "relu": torch.relu,
    }[s["activation"]]
    y = act(z[-1])
    if s["gated"]:
        y = y * z[0]
    if s["gate"] is not None:
        y = y * torch.index_select(s["gate"].double(), 0, s["index"])
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return _exact_8_bits(y) if s["quantize"] else y


_EXACT = {"quantize": _exact_quantize, "norm": _exact_norm, "linear": _exact_linear}


def exact(case: dict, seed: int):
    return _EXACT[case["op"]](prepare(case, seed))
