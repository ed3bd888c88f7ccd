"""Timed cases of the operators around a DiT block's attention and MLP, with their plain forms.

Every case is one pass through one operator:

* ``linear`` - ``fused_linear``: a matrix product whose epilogue adds the bias, applies the
  activation (or the gated activation over the two halves of the features), multiplies by the
  token's gate row and adds the residual;
* ``norm``   - ``fused_rmsnorm_residual_gate_rmsnorm_modulate``: the norm after a branch, its gate
  and (scaled) residual, the norm and modulation before the next branch;
* ``select`` - ``select_key_blocks``: the key blocks that the means of query and key blocks select;
* ``sparse`` - ``sparse_attn_func``: attention over such lists of key blocks.

The framework is inference only, so there is no backward direction. Activations are bf16; weights
of norms, biases and modulation tables bf16 or fp32.
"""

from __future__ import annotations

import math

import torch

own = False

D = 128
EPS = 1e-5
BLOCK_Q, BLOCK_K = 256, 64  # rows of a query block and of a key block
TABLE_ROWS = 9  # modulation rows of a block
MAX_FLOPS = 2 * 6240 * 5376 * 28672  # the largest listed case
MAX_BYTES = 2 * 6240 * (5376 + 14336) + 2 * 5376 * 28672


def listed() -> list[dict]:
    return [
        # The projection of one timestep's embedding: a single token, where the
        # weight rows and the call's own latency are all there is.
        _linear("linear_1_token", 1, 1024, 1024, activation="silu", bias="bf16"),
        # The modulation rows of a block (9 timestep rows, six vectors of the
        # hidden width each): bound by reading the weights.
        _linear("linear_modulation_rows", 9, 5376, 6 * 5376, bias="bf16"),
        # The audio segment's 1,296 tokens and one more through an odd-width
        # adapter with a GELU, back onto the residual: ragged in every tile.
        _linear("linear_ragged_gelu", 1297, 1544, 2056, activation="gelu_tanh", bias="f32", residual=True),
        # MLP up of one Ulysses rank at 480p / 5 s: the gated activation.
        _linear("mlp_up_rank", 6240, 5376, 14336, activation="silu", gated=True),
        # MLP down of the same rows, with the gated residual of the block.
        _linear("mlp_down_rank", 6240, 14336, 5376, bias="bf16", residual=True, gate="bf16"),
        # The norms around a branch at the microbenchmark's row count: latency.
        _norm("norm_257", 257, 5376, "bf16"),
        # The same on one rank's rows.
        _norm("norm_rank", 6240, 5376, "bf16"),
        # Block selection of a short joint sequence, one tenth of the keys kept.
        {"name": "select_frame_h40", "op": "select", "batch": 1, "sq": 1560, "sk": 1560, "heads": 40, "topk": 5, "always": 0},
        # Block selection of one head shard of a 480p / 5 s block; the blocks of
        # a text prefix are always kept.
        {"name": "select_480p_h5", "op": "select", "batch": 1, "sq": 49920, "sk": 49920, "heads": 5, "topk": 156, "always": 4},
        # A few query rows (a first frame's last tokens) against a long key
        # range: one query block a head.
        _sparse("sparse_16_rows", 1, 16, 12480, 8, 24),
        # A small sparse call: a quarter of 4,095 keys (the last block ragged).
        _sparse("sparse_4095_h4", 1, 4095, 4095, 4, 16),
        # One head shard of a 480p / 5 s block with a fifth of the keys kept.
        _sparse("sparse_480p_h5", 1, 49920, 49920, 5, 156),
    ]


def _linear(name, m, k, n, activation="none", gated=False, bias="none", residual=False, gate="none"):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "activation": activation, "gated": gated, "bias": bias,
            "residual": residual, "gate": gate}


def _norm(name, rows, cols, tables, weights="bf16", scaled=False):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "tables": tables, "weights": weights, "scaled": scaled}


def _sparse(name, batch, sq, sk, heads, topk, counts=False):
    return {"name": name, "op": "sparse", "batch": batch, "sq": sq, "sk": sk, "heads": heads, "topk": topk, "counts": counts}


def draw(rng) -> dict:
    """One more case: the same operators, sizes spread over their ranges."""

    def log_int(lo: int, hi: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "select", "sparse", "sparse"])
    if op == "linear":
        m = log_int(1, 64) if rng.random() < 0.35 else log_int(64, 12480)
        k, n = 8 * log_int(8, 1792), 8 * log_int(8, 1792)
        gated = rng.random() < 0.3
        while 2 * m * k * n * (1 + gated) > MAX_FLOPS:
            m = m // 2
        residual = not gated and rng.random() < 0.5
        case = _linear("", m, k, n, rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu"]), gated,
                       rng.choice(["none", "bf16", "f32"]), residual, rng.choice(["none", "bf16", "f32"]) if residual else "none")
    elif op == "norm":
        cols = rng.choice([1024, 2056, 5120, 5376, 6144, 1001]) if rng.random() < 0.6 else 8 * log_int(8, 1024)
        case = _norm("", log_int(1, 12480), cols, rng.choice(["bf16", "bf16", "f32"]), rng.choice(["bf16", "f32"]), rng.random() < 0.4)
    else:
        heads, batch = rng.choice([1, 2, 4, 5, 8, 10, 20, 40]), rng.choice([1, 1, 1, 2])
        sq = log_int(1, 49920)
        sk = sq if rng.random() < 0.6 else log_int(1, 49920)
        while batch * heads * (sq + sk) > 10 * 49920:
            heads, batch = max(1, heads // 2), 1
        nk = -(-sk // BLOCK_K)
        if op == "select":
            case = {"name": "", "op": op, "batch": batch, "sq": sq, "sk": sk, "heads": heads,
                    "topk": max(1, int(nk * rng.uniform(0.05, 0.5))), "always": rng.choice([0, 0, 1, 4])}
        else:
            topk = max(1, int(nk * rng.uniform(0.03, 0.5)))
            while 4 * D * batch * heads * sq * topk * BLOCK_K > MAX_FLOPS:
                topk = topk // 2
            case = _sparse("", batch, sq, sk, heads, topk, rng.random() < 0.4)
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

    def gain(self, n: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return (1.0 + self.normal(n, dtype=torch.float32, scale=0.1)).to(dtype)

    def index(self, rows: int) -> torch.Tensor:
        """The modulation row of each token: frames in order."""
        return torch.arange(rows, device=self.device) * TABLE_ROWS // max(rows, 1)

    def heads_normed(self, batch: int, seq: int, heads: int, share: torch.Tensor) -> torch.Tensor:
        """q or k as attention meets them: RMS-normalised per head, with a part
        that neighbouring tokens share (``share``: one vector per 52 tokens)."""
        x = torch.randn((batch, seq, heads, D), device=self.device, generator=self.generator)
        x += share[:, torch.arange(seq, device=self.device) // 52 % share.shape[1]]
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).to(torch.bfloat16)

    def qk(self, batch: int, sq: int, sk: int, heads: int) -> tuple[torch.Tensor, torch.Tensor]:
        share = torch.randn((batch, 1 + max(sq, sk) // 52, heads, D), device=self.device, generator=self.generator)
        return self.heads_normed(batch, sq, heads, share), self.heads_normed(batch, sk, heads, share)

    def lists(self, batch: int, heads: int, nq: int, nk: int, topk: int) -> torch.Tensor:
        """Key-block lists as selection gives them: the blocks near the query's
        own, some that all queries of a head look at, others by chance."""
        score = torch.rand((batch, heads, nq, nk), device=self.device, generator=self.generator)
        score += 0.5 * torch.rand((batch, heads, 1, nk), device=self.device, generator=self.generator)
        own_block = torch.arange(nq, device=self.device)[:, None] * (nk / max(nq, 1))
        score += (own_block - torch.arange(nk, device=self.device)).abs() < 3
        return score.topk(topk, dim=-1).indices.sort(dim=-1).values.to(torch.int32)


_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case: dict, seed: int) -> dict:
    rng = _Inputs(seed)
    op = case["op"]
    s: dict = {"op": op}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        rows = 2 * n if case["gated"] else n
        s["x"] = rng.normal(m, k)
        s["weight"] = rng.normal(rows, k, scale=k**-0.5)
        s["bias"] = None if case["bias"] == "none" else rng.normal(rows, dtype=_DTYPES[case["bias"]], scale=0.1)
        s["activation"] = None if case["activation"] == "none" else case["activation"]
        s["gated"] = case["gated"]
        s["residual"] = rng.normal(m, n, scale=2.0) if case["residual"] else None
        s["gate"] = s["index"] = None
        if case["gate"] != "none":
            # one of the six modulation vectors that lie side by side in a row
            s["gate"] = rng.normal(TABLE_ROWS, 3 * n, dtype=_DTYPES[case["gate"]], scale=0.3).chunk(3, dim=-1)[2]
            s["index"] = rng.index(m)
    elif op == "norm":
        rows, cols = case["rows"], case["cols"]
        s["branch"], s["residual"] = rng.normal(1, rows, cols), rng.normal(1, rows, cols, scale=2.0)
        s["branch_weight"], s["weight"] = (rng.gain(cols, _DTYPES[case["weights"]]) for _ in range(2))
        tables = rng.normal(TABLE_ROWS, 3 * cols, dtype=_DTYPES[case["tables"]], scale=0.3)
        s["shift"], s["scale"], s["gate"] = tables.chunk(3, dim=-1)
        s["index"] = rng.index(rows)
        s["residual_scale"] = 0.75 if case["scaled"] else 1.0
    elif op == "select":
        s["q"], s["k"] = rng.qk(case["batch"], case["sq"], case["sk"], case["heads"])
        s["topk"] = case["topk"]
        nk = -(-case["sk"] // BLOCK_K)
        s["always"] = torch.arange(nk, device=rng.device) < case["always"] if case["always"] else None
    else:
        b, sq, sk, h = case["batch"], case["sq"], case["sk"], case["heads"]
        s["q"], s["k"] = rng.qk(b, sq, sk, h)
        s["v"] = rng.normal(b, sk, h, D)
        nq, nk = -(-sq // BLOCK_Q), -(-sk // BLOCK_K)
        s["block_index"], s["block_count"] = rng.lists(b, h, nq, nk, case["topk"]), None
        if case["counts"]:
            s["block_count"] = torch.randint(0, case["topk"] + 1, (b, h, nq), device=rng.device, generator=rng.generator).to(torch.int32)
    return s


# ---------------------------------------------------------------- plain forms, 32 bits


def _activate(z: torch.Tensor, kind: str | None) -> torch.Tensor:
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5**0.5))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z * (z > 0) if kind == "relu" else z


def _plain_linear(s: dict) -> torch.Tensor:
    z = s["x"].float() @ s["weight"].float().t()
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
    return y.to(torch.bfloat16)


def _plain_norm(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    t = s["index"]
    gate, scale, shift = (s[n].float()[t] for n in ("gate", "scale", "shift"))
    x = s["branch"].float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["branch_weight"].float()
    h = s["residual_scale"] * s["residual"].float() + gate * x
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float() * (1.0 + scale) + shift
    return h.to(torch.bfloat16), y.to(torch.bfloat16)


def _block_means(x: torch.Tensor, block: int) -> torch.Tensor:
    """(B, S, H, D) -> (B, H, blocks, D): sums in 64 bits, means rounded to 32
    (the order of scores next to each other is the operator's result)."""
    b, n, h, d = x.shape
    blocks = -(-n // block)
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, 0, 0, blocks * block - n)).view(b, blocks, block, h, d).sum(2)
    rows = torch.full((blocks,), block, dtype=torch.float64, device=x.device)
    rows[-1] = n - (blocks - 1) * block
    return (x / rows[:, None, None]).float().permute(0, 2, 1, 3).contiguous()


def _plain_select(s: dict) -> torch.Tensor:
    qm, km = _block_means(s["q"], BLOCK_Q).double(), _block_means(s["k"], BLOCK_K).double()
    score = torch.matmul(qm, km.transpose(-1, -2).contiguous()).float()
    if s["always"] is not None:
        score = torch.where(s["always"], float("inf"), score)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    return order[..., : min(s["topk"], score.shape[-1])].sort(dim=-1).values.to(torch.int32)


def _plain_sparse(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    q, index, count = s["q"], s["block_index"].long(), s["block_count"]
    b, sq, h, _ = q.shape
    sk, nk, topk = s["k"].shape[1], -(-s["k"].shape[1] // BLOCK_K), index.shape[-1]
    grow = (0, 0, 0, 0, 0, nk * BLOCK_K - sk)
    k, v = (torch.nn.functional.pad(s[n].float(), grow).permute(0, 2, 1, 3).reshape(b * h, nk, BLOCK_K * D) for n in "kv")
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
    heads = torch.arange(b * h, device=q.device)[:, None]
    position = torch.arange(BLOCK_K, device=q.device)
    for i in range(index.shape[2]):
        rows = slice(i * BLOCK_Q, min((i + 1) * BLOCK_Q, sq))
        ids = index[:, :, i].reshape(b * h, topk)
        keep = (ids[..., None] * BLOCK_K + position) < sk
        if count is not None:
            keep = keep & (torch.arange(topk, device=q.device) < count[:, :, i].reshape(b * h, 1))[..., None]
        qi = q[:, rows].float().permute(0, 2, 1, 3).reshape(b * h, -1, D)
        x = torch.matmul(qi, k[heads, ids].view(b * h, topk * BLOCK_K, D).transpose(-1, -2).contiguous()) / math.sqrt(D)
        x = x.masked_fill(~keep.view(b * h, 1, topk * BLOCK_K), float("-inf"))
        top = x.amax(-1, keepdim=True)
        x = torch.exp(x - top.clamp_min(-3.0e38))
        total = x.sum(-1, keepdim=True)
        o = torch.matmul(x, v[heads, ids].view(b * h, topk * BLOCK_K, D)) / total.clamp_min(1.0e-37)
        out[:, rows] = o.view(b, h, -1, D).permute(0, 2, 1, 3).to(torch.bfloat16)
        lse[:, :, rows] = (top + total.log()).view(b, h, -1)
    return out, lse


_PLAIN = {"linear": _plain_linear, "norm": _plain_norm, "select": _plain_select, "sparse": _plain_sparse}


def _own(s: dict):
    op = s["op"]
    if op == "linear":
        from h3_flash_amd import fused_linear

        return fused_linear(s["x"], s["weight"], s["bias"], activation=s["activation"], gated=s["gated"],
                            residual=s["residual"], gate=s["gate"], index=s["index"])
    if op == "norm":
        from h3_flash_amd.fusions import fused_rmsnorm_residual_gate_rmsnorm_modulate

        return fused_rmsnorm_residual_gate_rmsnorm_modulate(
            s["residual"], s["branch"], s["branch_weight"], s["gate"], s["weight"], s["scale"], s["shift"], s["index"], EPS,
            residual_scale=s["residual_scale"],
        )
    if op == "select":
        from h3_flash_amd import select_key_blocks

        return select_key_blocks(s["q"], s["k"], s["topk"], always=s["always"])
    from h3_flash_amd import sparse_attn_func

    return sparse_attn_func(s["q"], s["k"], s["v"], s["block_index"], s["block_count"])


def run(s: dict):
    return _own(s) if own else _PLAIN[s["op"]](s)


def work(case: dict) -> dict:
    op = case["op"]
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        rows = 2 * n if case["gated"] else n
        size = {"none": 0, "bf16": 2, "f32": 4}
        nbytes = 2 * (m * k + rows * k + m * n * (2 if case["residual"] else 1)) + size[case["bias"]] * rows
        if case["gate"] != "none":
            nbytes += size[case["gate"]] * TABLE_ROWS * n + 8 * m
        flops = 2 * m * k * rows
    elif op == "norm":
        n = case["rows"] * case["cols"]
        size = {"bf16": 2, "f32": 4}
        nbytes = 8 * n + case["cols"] * (3 * TABLE_ROWS * size[case["tables"]] + 2 * size[case["weights"]]) + 8 * case["rows"]
        flops = 14 * n
    else:
        b, sq, sk, h = case["batch"], case["sq"], case["sk"], case["heads"]
        nq, nk = -(-sq // BLOCK_Q), -(-sk // BLOCK_K)
        if op == "select":
            nbytes = 2 * D * b * h * (sq + sk) + 4 * b * h * nq * min(case["topk"], nk)
            flops = b * h * D * (2 * nq * nk + sq + sk)
        else:
            # by the mean length where rows name fewer blocks than the list holds
            blocks = case["topk"] / (2 if case["counts"] else 1)
            keys = min(blocks * BLOCK_K, sk)
            nbytes = b * h * (sq * (4 * D + 4) + int(min(nq * keys, sk)) * 4 * D + 4 * nq * case["topk"])
            flops = int(4 * D * b * h * sq * keys)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------- 64 bits


def _exact_linear(s: dict) -> torch.Tensor:
    z = torch.nn.functional.linear(s["x"].double(), s["weight"].double(), None if s["bias"] is None else s["bias"].double())
    kind = s["activation"]
    act = {
        None: lambda a: a,
        "silu": lambda a: a * torch.sigmoid(a),
        "gelu": lambda a: torch.nn.functional.gelu(a),
        "gelu_tanh": lambda a: torch.nn.functional.gelu(a, approximate="tanh"),
        "relu": torch.relu,
    }[kind]
    half = z.shape[1] // 2
    y = z[:, :half] * act(z[:, half:]) if s["gated"] else act(z)
    if s["gate"] is not None:
        y = y * torch.index_select(s["gate"].double(), 0, s["index"])
    return y if s["residual"] is None else s["residual"].double() + y


def _exact_norm(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    cols = (s["branch"].shape[-1],)
    gate, scale, shift = (torch.index_select(s[n].double(), 0, s["index"]) for n in ("gate", "scale", "shift"))
    post = torch.nn.functional.rms_norm(s["branch"].double(), cols, s["branch_weight"].double(), EPS)
    hidden = s["residual"].double() * s["residual_scale"] + gate * post
    normed = torch.nn.functional.rms_norm(hidden, cols, s["weight"].double(), EPS)
    return hidden, normed * (scale + 1.0) + shift


def _exact_select(s: dict) -> torch.Tensor:
    q, k = s["q"].double(), s["k"].double()
    b, _, h, _ = q.shape
    means = []
    for x, block in ((q, BLOCK_Q), (k, BLOCK_K)):
        means.append(torch.stack([part.mean(dim=1) for part in x.split(block, dim=1)], dim=2).float().double())
    rows = []
    for i in range(b):
        for j in range(h):
            score = (means[0][i, j] @ means[1][i, j].t()).float().double()
            if s["always"] is not None:
                score[:, s["always"]] = float("inf")
            # the rank of a block: how many come before it
            place = torch.empty(score.shape, dtype=torch.int64, device=score.device)
            order = torch.argsort(-score, dim=-1, stable=True)
            place.scatter_(1, order, torch.arange(score.shape[1], device=score.device).expand_as(order).contiguous())
            kept = place < s["topk"]
            rows.append(kept.nonzero()[:, 1].view(score.shape[0], -1))
    return torch.stack(rows).view(b, h, rows[0].shape[0], -1).to(torch.int32)


def _exact_sparse(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    b, sq, h, _ = s["q"].shape
    sk = s["k"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((b, h, sq), float("-inf"), dtype=torch.float64, device=out.device)
    counts = None if s["block_count"] is None else s["block_count"].tolist()
    within = torch.arange(BLOCK_K, device=out.device)
    for i in range(b):
        for j in range(h):
            q, k, v = (s[n][i, :, j].double() for n in "qkv")
            for t in range(s["block_index"].shape[2]):
                ids = s["block_index"][i, j, t].long()
                if counts is not None:
                    ids = ids[: counts[i][j][t]]
                keys = (ids[:, None] * BLOCK_K + within).flatten()
                if int(ids.numel()) == 0:
                    continue
                at = slice(t * BLOCK_Q, (t + 1) * BLOCK_Q)
                past = keys >= sk
                keys = keys.clamp_max(sk - 1)
                x = (q[at] @ k[keys].t()) * D**-0.5
                x = torch.where(past, float("-inf"), x)
                l = torch.logsumexp(x, dim=-1)
                out[i, at, j] = torch.exp(x - l[:, None]) @ v[keys]
                lse[i, j, at] = l
    return out, lse


_EXACT = {"linear": _exact_linear, "norm": _exact_norm, "select": _exact_select, "sparse": _exact_sparse}


def exact(case: dict, seed: int):
    return _EXACT[case["op"]](prepare(case, seed))
