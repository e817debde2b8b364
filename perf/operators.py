"""Cases of the 8-bit block operators: activation checkpoints, products and the feed-forward half of a block.

A matrix is held in 8 bits as e4m3 values with one power-of-two scale for each block: 128 neighbouring values of one row
(``rows`` = 1: what one token is stored as does not depend on its neighbours) or a tile of 128 rows by 128 columns
(``rows`` = 128: the same bytes serve a product over the columns and one over the rows).  The scale of a block is the
smallest power of two, from 2^-127 up, that brings the block's largest magnitude to at most 448; values are rounded to
the nearest e4m3 number, ties to even.  Weights are always held in tiles.

Operators (``op`` of a case):

* ``checkpoint``      pack an activation and read it back;
* ``linear``          ``x W^T`` of packed operands; ``frozen``: the weight was packed beforehand and ``x`` is packed row by
                      row, else both are packed in the call, in tiles.  With ``grad`` also the gradients, whose incoming
                      gradient is packed like ``x``;
* ``ffn``             ``residual + h W_v^T``, ``h = relu(xk W_k^T)^2`` kept in 8 bits; its backward pass reads that ``h``.
"""
import math

import torch

own = False

OUTLIERS = 64          # one channel in 64 of an activation is far larger than the others, as in a trained residual stream


def listed():
    return [
        # one chunk of infinite-context training of the 0.4B network: the input of one recomputed block
        {"name": "checkpoint of a chunk", "op": "checkpoint", "tokens": 512, "width": 1024, "rows": 1, "dtype": "bf16"},
        # the headline pre-training micro-batch of the 1.5B network (8 x 4096 tokens)
        {"name": "checkpoint of a batch", "op": "checkpoint", "tokens": 32768, "width": 2048, "rows": 1, "dtype": "bf16"},
        # a ragged fine-tuning batch kept in tiles, from an fp32 run, with widths that end inside a block
        {"name": "checkpoint, ragged tiles", "op": "checkpoint", "tokens": 4099, "width": 1990, "rows": 128, "dtype": "fp32"},
        # one generated token, a square projection
        {"name": "linear, one token", "op": "linear", "tokens": 1, "width": 2048, "out": 2048, "frozen": True, "grad": False},
        # the vocabulary head of a rollout step of 64 sequences
        {"name": "linear, head of 64", "op": "linear", "tokens": 64, "width": 2048, "out": 65536, "frozen": True, "grad": False},
        # adapter training over a frozen 2.9B projection: output and input gradient
        {"name": "linear, frozen", "op": "linear", "tokens": 4096, "width": 2560, "out": 2560, "frozen": True, "grad": True},
        # a short odd batch through a map whose sides are no multiple of a block
        {"name": "linear, odd", "op": "linear", "tokens": 1001, "width": 1000, "out": 523, "frozen": False, "grad": True},
        # a full-parameter projection of the headline step
        {"name": "linear, training", "op": "linear", "tokens": 32768, "width": 2048, "out": 2048, "frozen": False, "grad": True},
        # feed-forward half for one generated token
        {"name": "ffn, one token", "op": "ffn", "tokens": 1, "width": 2048, "hidden": 8192, "frozen": True, "grad": False},
        # the same for a rollout of 64 sequences
        {"name": "ffn, rollout of 64", "op": "ffn", "tokens": 64, "width": 2048, "hidden": 8192, "frozen": True, "grad": False},
        # ragged fine-tuning batch of the 0.4B network
        {"name": "ffn, ragged training", "op": "ffn", "tokens": 1111, "width": 1024, "hidden": 4096, "frozen": False, "grad": True},
        # the headline step's feed-forward half
        {"name": "ffn, training", "op": "ffn", "tokens": 32768, "width": 2048, "hidden": 8192, "frozen": False, "grad": True},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["checkpoint", "linear", "linear", "ffn", "ffn"])
    if op == "checkpoint":
        width = _between(rng, 64, 8192)
        return {"op": op, "tokens": _between(rng, 1, min(32768, 2 ** 26 // width)), "width": width, "rows": rng.choice([1, 128]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    frozen = rng.random() < 0.6
    grad = True if not frozen else rng.random() < 0.4
    width = _between(rng, 64, 4096)
    if rng.random() < 0.6:
        width = max(64, width // 64 * 64)          # most networks have whole heads; the others end inside a block
    tokens = _between(rng, 1, 128) if frozen and not grad and rng.random() < 0.5 else _between(rng, 1, 32768)
    if op == "linear":
        out = _between(rng, 16, 16384)
        tokens = min(tokens, max(1, 2 ** 38 // (width * out)))
        return {"op": op, "tokens": tokens, "width": width, "out": out, "frozen": frozen, "grad": grad}
    hidden = 4 * width
    tokens = min(tokens, max(1, 2 ** 38 // (width * hidden)))
    return {"op": op, "tokens": tokens, "width": width, "hidden": hidden, "frozen": frozen, "grad": grad}


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(case, seed):
    """The tensors of a case, made on the GPU from the seed alone."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(1000003 * (seed + 1))
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    t, c = case["tokens"], case["width"]

    def activation(rows, cols, dtype):
        a = rnd(rows, cols)
        a[:, torch.randint(0, cols, (max(1, cols // OUTLIERS),), generator=g, device=dev)] *= 20.0
        return a.to(dtype)

    def weight(n, k):
        return (torch.rand(n, k, generator=g, device=dev) - 0.5).mul_(2.0 / math.sqrt(k)).to(torch.bfloat16)

    def gradient(rows, cols):       # token losses differ by orders of magnitude
        return rnd(rows, cols).mul_(torch.exp(1.5 * rnd(rows, 1)) / rows).to(torch.bfloat16)

    if case["op"] == "checkpoint":
        return {"x": activation(t, c, _TYPES[case["dtype"]])}
    s = {"x": activation(t, c, torch.bfloat16)}
    if case["op"] == "linear":
        s["w"] = weight(case["out"], c)
        if case["grad"]:
            s["dy"] = gradient(t, case["out"])
        return s
    s.update(wk=weight(case["hidden"], c), wv=weight(c, case["hidden"]), residual=activation(t, c, torch.bfloat16))
    if case["grad"]:
        s["dy"] = gradient(t, c)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] != "checkpoint" and case["frozen"]:        # a frozen weight is packed once and kept in that form
        for name in [n for n in ("w", "wk", "wv") if n in s]:
            if own:
                from rwkvtune_b200 import ops

                s[name] = ops.pack_fp8(s[name], rows=128)
            else:
                s[name] = _packed(s[name], 128)
    elif case["op"] != "checkpoint" and case["grad"]:
        for name in [n for n in ("w", "wk", "wv") if n in s]:
            s[name].requires_grad_(True)
    if case.get("grad"):
        s["x"].requires_grad_(True)
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from rwkvtune_b200 import ops

    case = s["case"]
    if case["op"] == "checkpoint":
        return ops.unpack_fp8(ops.pack_fp8(s["x"], rows=case["rows"]))
    if not case["grad"]:
        with torch.no_grad():
            if case["op"] == "linear":
                return ops.fp8_linear(s["x"], s["w"])
            return ops.fp8_channel_mix_ffn(s["x"], s["wk"], s["wv"], s["residual"])
    if case["op"] == "linear":
        y = ops.fp8_linear(s["x"], s["w"])
        names = ["x"] if case["frozen"] else ["x", "w"]
    else:
        y = ops.fp8_channel_mix_ffn(s["x"], s["wk"], s["wv"], s["residual"])
        names = ["x"] if case["frozen"] else ["x", "wk", "wv"]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


# ---------------------------------------------------------------------------------------------- the plain form
def _power(n):
    """2^n in fp32 for whole n from -127 on (two factors, each a normal number)."""
    half = torch.div(n, 2, rounding_mode="floor")
    return ((half + 127) << 23).view(torch.float32) * ((n - half + 127) << 23).view(torch.float32)


def _packed(x, rows):
    """The fp32 values that ``x`` stands for once it is packed in blocks of ``rows`` by 128."""
    x = x.detach().float()
    m, k = x.shape
    padded = torch.zeros(-(-m // rows) * rows, -(-k // 128) * 128, device=x.device)
    padded[:m, :k] = x
    blocks = padded.view(padded.shape[0] // rows, rows, padded.shape[1] // 128, 128)
    largest = blocks.abs().amax(dim=(1, 3), keepdim=True)
    part, power = torch.frexp(largest)                         # largest = part * 2^power, part in [0.5, 1)
    shift = torch.where(part > 0.875, power - 8, power - 9)    # 448 = 0.875 * 2^9
    shift = torch.where(largest > 0, shift, -127).clamp(min=-127).to(torch.int32)
    v = blocks * _power(-shift)
    _, power = torch.frexp(v)
    step = _power((power - 1).clamp(min=-6).to(torch.int32) - 3)   # distance of e4m3 numbers around v
    v = torch.round(v / step) * step * _power(shift)
    return v.view(padded.shape)[:m, :k]


def _run_plain(s):
    case = s["case"]
    bf = torch.bfloat16
    with torch.no_grad():
        if case["op"] == "checkpoint":
            return _packed(s["x"], case["rows"]).to(s["x"].dtype)
        rows = 1 if case["frozen"] else 128
        held = (lambda w: w) if case["frozen"] else (lambda w: _packed(w, 128))
        x = _packed(s["x"], rows)
        if case["op"] == "linear":
            w = held(s["w"])
            y = (x @ w.t()).to(bf)
            if not case["grad"]:
                return y
            d = _packed(s["dy"], rows)
            out = {"y": y, "dx": (d @ w).to(bf)}
            if not case["frozen"]:
                out["dw"] = (d.t() @ x).to(bf)
            return out
        wk, wv = held(s["wk"]), held(s["wv"])
        h = _packed(torch.relu(x @ wk.t()) ** 2, rows)
        y = (s["residual"].float() + h @ wv.t()).to(bf)
        if not case["grad"]:
            return y
        d = _packed(s["dy"], rows)
        p = _packed((d @ wv) * 2 * torch.sqrt(h), rows)
        out = {"y": y, "dx": (p @ wk).to(bf)}
        if not case["frozen"]:
            out["dwk"], out["dwv"] = (p.t() @ x).to(bf), (d.t() @ h).to(bf)
        return out


# ---------------------------------------------------------------------------------------------- 64 bits, written apart
def _exact_packed(x, rows):
    """Packing by its definition: candidate scales are compared with the largest magnitude, and each value takes the
    nearest entry of the list of e4m3 numbers."""
    x = x.detach().double()
    dev = x.device
    numbers = [i * 2.0 ** -9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 3) for e in range(-6, 9) for i in range(8)][:-1]
    numbers = torch.tensor(numbers, dtype=torch.float64, device=dev)          # entry i has the bit pattern i
    halves = (numbers[1:] + numbers[:-1]) / 2
    scales = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64, device=dev)
    out = torch.empty_like(x)
    m, k = x.shape
    for top in range(0, m, 8192):                                             # 8192 rows at a time: memory
        part = x[top:top + 8192]
        pad_rows, pad_cols = -part.shape[0] % rows, -k % 128
        p = torch.nn.functional.pad(part, (0, pad_cols, 0, pad_rows))
        p = p.unflatten(1, (-1, 128)).unflatten(0, (-1, rows)).movedim(1, 2)  # [row block, column block, rows, 128]
        largest = p.abs().flatten(2).max(dim=2).values
        scale = scales[torch.searchsorted(scales * 448.0, largest.contiguous())][..., None, None]
        v = p / scale
        mag = v.abs().contiguous()
        at = torch.searchsorted(halves, mag)                                  # number of half-way points below mag
        tie = (at < halves.numel()) & (halves[at.clamp(max=halves.numel() - 1)] == mag) & (at % 2 == 1)
        v = torch.copysign(numbers[at + tie.long()], v) * scale
        out[top:top + 8192] = v.movedim(2, 1).flatten(2, 3).flatten(0, 1)[:part.shape[0], :k]
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        if case["op"] == "checkpoint":
            return _exact_packed(s["x"], case["rows"])
        if not torch.cuda.is_available() and case["tokens"] * case["width"] * case.get("out", 4 * case["width"]) > 2 ** 33:
            return None
        rows = 1 if case["frozen"] else 128
        x = _exact_packed(s["x"], rows)
        if case["op"] == "linear":
            w = _exact_packed(s["w"], 128)
            y = torch.einsum("mk,nk->mn", x, w)
            if not case["grad"]:
                return y
            d = _exact_packed(s["dy"], rows)
            out = {"y": y, "dx": torch.einsum("mn,nk->mk", d, w)}
            if not case["frozen"]:
                out["dw"] = torch.einsum("mn,mk->nk", d, x)
            return out
        wk, wv = _exact_packed(s["wk"], 128), _exact_packed(s["wv"], 128)
        a = torch.einsum("mk,nk->mn", x, wk)
        h = _exact_packed(torch.where(a > 0, a * a, torch.zeros_like(a)), rows)
        y = s["residual"].double() + torch.einsum("mn,kn->mk", h, wv)
        if not case["grad"]:
            return y
        d = _exact_packed(s["dy"], rows)
        p = _exact_packed(2 * h.sqrt() * torch.einsum("mk,kn->mn", d, wv), rows)
        out = {"y": y, "dx": torch.einsum("mn,nk->mk", p, wk)}
        if not case["frozen"]:
            out["dwk"] = torch.einsum("mn,mk->nk", p, x)
            out["dwv"] = torch.einsum("mk,mn->kn", d, h)
        return out


def work(case):
    t, c = case["tokens"], case["width"]
    if case["op"] == "checkpoint":      # read, the 8-bit form written and read, written
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": t * c * (2 * size + 2), "flops": 0}
    n = case["out"] if case["op"] == "linear" else case["hidden"]
    weight = n * c * (1 if case["frozen"] else 2)              # 8-bit weights are read as such
    products = 1 if not case["grad"] else 2 if case["frozen"] else 3
    if case["op"] == "linear":
        moved = 2 * t * (c + n) + weight
        if case["grad"]:
            moved += 2 * t * (c + n) + (0 if case["frozen"] else 2 * n * c)
        return {"bytes": moved, "flops": 2 * t * n * c * products}
    moved = 2 * t * 3 * c + 2 * weight
    if case["grad"]:
        moved += 2 * t * 2 * c + (0 if case["frozen"] else 4 * n * c)
    return {"bytes": moved, "flops": 2 * 2 * t * n * c * products}
