"""Cases that measure the 8-bit operators of elips_b200.int8: matrix products of int8 codes with a scale per row
and channel, the layer that quantises its input rows first, and the paged cache that quantises rows as they are
written and gives them back."""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # One query against 10,000 stored rows: the latency of a single product.
        {"name": "scores of one query", "kind": "gemm", "m": 1, "n": 10000, "k": 768, "out": "fp32", "bias": "", "pitch": 16},
        # A batch of queries against a base of rows, every score kept.
        {"name": "scores of 64 queries", "kind": "gemm", "m": 64, "n": 100000, "k": 384, "out": "fp32", "bias": "", "pitch": 16},
        # Sizes that fit no tile, rows that start anywhere.
        {"name": "odd product", "kind": "gemm", "m": 333, "n": 1001, "k": 1111, "out": "fp16", "bias": "fp32", "pitch": 1},
        # The tokens of a batch of prompts through one projection.
        {"name": "projection", "kind": "gemm", "m": 4096, "n": 4096, "k": 4096, "out": "bf16", "bias": "bf16", "pitch": 16},
        # A large square product, bound by the matrix instructions.
        {"name": "large product", "kind": "gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "bias": "", "pitch": 16},
        # One token through a layer while it is being generated.
        {"name": "layer, one token", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": ""},
        # One token for each of a few sequences.
        {"name": "layer, 24 tokens", "kind": "linear", "m": 24, "n": 6144, "k": 1536, "type": "fp16", "bias": "fp16"},
        # 10,000 embeddings through an adapter to twice their width.
        {"name": "layer, 10,000 rows", "kind": "linear", "m": 10000, "n": 1536, "k": 768, "type": "fp32", "bias": "fp32"},
        # A few sequences, one new token each: written, and the short contexts read back.
        {"name": "cache, new tokens", "kind": "cache", "parts": 2, "sequences": 4, "longest": 40, "new": 1, "heads": 8,
         "dim": 128, "page": 16, "type": "bf16", "padding": 0},
        # Prompts of different lengths written whole and read back, with padding rows in the batch.
        {"name": "cache, prompts", "kind": "cache", "parts": 2, "sequences": 6, "longest": 4096, "new": 4096, "heads": 8,
         "dim": 128, "page": 16, "type": "bf16", "padding": 37},
        # One long context read back.
        {"name": "read, long context", "kind": "read", "parts": 2, "sequences": 1, "longest": 131072, "heads": 8,
         "dim": 128, "page": 64, "type": "bf16"},
        # Vectors of many documents, one head, a width that ends inside a vector of bytes.
        {"name": "read, many documents", "kind": "read", "parts": 1, "sequences": 300, "longest": 180, "heads": 1,
         "dim": 388, "page": 32, "type": "fp16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _odd(rng, value, step):
    """`value` as it is half of the time, else the multiple of `step` below it."""
    return value if rng.random() < 0.5 or value < step else value // step * step


def draw(rng):
    kind = rng.choice(["gemm", "gemm", "linear", "linear", "cache", "read"])
    if kind in ("gemm", "linear"):
        k = _odd(rng, _log(rng, 32, 16384), 64)
        n = _odd(rng, _log(rng, 16, 32768), 16)
        m = _odd(rng, _log(rng, 1, max(1, min(8192, 2 ** 38 // (n * k), 2 ** 26 // n))), 8)
        c = {"kind": kind, "m": m, "n": n, "k": k, "bias": rng.choice(["", "fp32", "bf16"])}
        if kind == "gemm":
            return {**c, "out": rng.choice(["fp32", "fp16", "bf16"]), "pitch": rng.choice([16, 16, 1])}
        return {**c, "type": rng.choice(["fp32", "fp16", "bf16"])}
    heads = rng.choice([1, 2, 3, 4, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 200, 256, 67]) if heads > 1 else _odd(rng, _log(rng, 32, 1536), 8)
    parts = rng.choice([1, 2])
    sequences = _log(rng, 1, 256)
    longest = _log(rng, 1, max(1, min(100000, 2 ** 26 // (sequences * heads * dim * parts))))
    c = {"kind": kind, "parts": parts, "sequences": sequences, "longest": longest, "heads": heads, "dim": dim,
         "page": rng.choice([1, 16, 32, 64, 128]), "type": rng.choice(["fp32", "fp16", "bf16"])}
    if kind == "cache":
        c |= {"new": rng.choice([1, 1, longest]), "padding": rng.choice([0, rng.randint(1, 64)])}
    return c


def _lengths(case):
    """The sequences' lengths: the same for every seed, the first the longest."""
    rng = random.Random(case["sequences"] * 1000003 + case["longest"])
    return [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(case["sequences"] - 1)]


def _activations(shape, gen):
    """Rows as a model's layers give them: unit normal with a few channels far larger, rows of different size."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    return x * torch.exp(torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))


def _codes(rows, width, pitch, gen):
    """int8 codes [rows, width] whose rows start on multiples of `pitch` bytes."""
    wide = -(-width // pitch) * pitch
    c = (torch.randn((rows, wide), generator=gen, device="cuda") * 40).round_().clamp_(-127, 127).to(torch.int8)
    return c[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        s["b"] = _codes(n, k, case.get("pitch", 16), gen)
        s["b_scales"] = torch.rand(n, generator=gen, device="cuda") * 1e-3 + 1e-4
        s["bias"] = torch.randn(n, generator=gen, device="cuda").to(TYPES[case["bias"]]) if case["bias"] else None
        if case["kind"] == "gemm":
            s["a"] = _codes(m, k, case["pitch"], gen)
            s["a_scales"] = torch.rand(m, generator=gen, device="cuda") * 0.05 + 1e-3
            s["type"] = TYPES[case["out"]]
        else:
            s["type"] = TYPES[case["type"]]
            s["x"] = _activations((m, k), gen).to(s["type"])
        return s
    parts, heads, dim, page = case["parts"], case["heads"], case["dim"], case["page"]
    lengths = _lengths(case)
    need = [-(-v // page) for v in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")[:sum(need)]
    at = torch.arange(max(need), device="cuda")[None, :]
    counts = torch.tensor(need, device="cuda")[:, None]
    table = torch.full((len(need), max(need)), -1, dtype=torch.int64, device="cuda")
    table[at < counts] = order
    s["page_table"] = table.to(torch.int32)
    ends = torch.tensor(lengths, device="cuda").cumsum(0)
    s["offsets"] = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    s["total"] = sum(lengths)
    s["type"] = TYPES[case["type"]]
    # The cache as it stands before the call: rows of 16-byte pitch, all of them holding earlier tokens.
    wide = -(-dim // 16) * 16
    codes = torch.randint(-127, 128, (parts, pages, page, heads, wide), generator=gen, device="cuda", dtype=torch.int8)
    s["codes"] = codes[..., :dim]
    s["scales"] = torch.rand((parts, pages, page, heads), generator=gen, device="cuda") * 0.05 + 1e-3
    if case["kind"] == "cache":
        seq = torch.cat([torch.full((min(case["new"], v),), i) for i, v in enumerate(lengths)]).cuda()
        pos = torch.cat([torch.arange(v - min(case["new"], v), v) for v in lengths]).cuda()
        slots = table[seq, pos // page] * page + pos % page
        s["slots"] = torch.cat([slots, slots.new_full((case["padding"],), -1)])
        s["rows"] = tuple(_activations((s["slots"].numel(), heads, dim), gen).to(s["type"]) for _ in range(parts))
    return s


def _quantise(x):
    """Codes and scale of each row (the last axis), as floats. The quotient is taken in 64 bits: it decides between
    neighbouring codes."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, torch.zeros_like(scale), scale)
    codes = torch.round(x.double() / scale.double()).float()
    return torch.where((scale > 0) & torch.isfinite(scale), codes, torch.zeros_like(codes)), scale


def _product(a, b, a_scales, b_scales, bias, dtype):
    out = (a @ b.t()) * a_scales[:, None] * b_scales
    return (out if bias is None else out + bias.float()).to(dtype)


def _write(s):
    codes, scales = s["codes"].flatten(1, 2), s["scales"].view(s["scales"].shape[0], -1, s["scales"].shape[3])
    slots, rows = s["slots"], torch.stack(s["rows"])
    if s["case"]["padding"]:
        kept = slots >= 0
        slots, rows = slots[kept], rows[:, kept]
    q, scale = _quantise(rows)
    codes[:, slots] = q.to(torch.int8)
    scales[:, slots] = scale[..., 0]


def _read(s):
    page = s["case"]["page"]
    t = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["offsets"][1:], t, right=True)
    pos = t - s["offsets"][seq]
    slots = s["page_table"][seq, pos // page].long() * page + pos % page
    codes, scales = s["codes"].flatten(1, 2), s["scales"].flatten(1, 2)
    return tuple((codes[:, slots].float() * scales[:, slots][..., None]).to(s["type"]).unbind(0))


def run(s):
    kind = s["kind"]
    if own:
        from elips_b200 import int8
        if kind == "gemm":
            return int8.gemm_int8(s["a"], s["b"], s["a_scales"], s["b_scales"], s["bias"], out_dtype=s["type"])
        if kind == "linear":
            return int8.linear_int8(s["x"], s["b"], s["b_scales"], s["bias"])
        if kind == "cache":
            int8.cache_write(s["codes"], s["scales"], s["rows"], s["slots"])
        return int8.cache_read(s["codes"], s["scales"], s["page_table"], s["offsets"], s["total"], s["type"])
    if kind == "gemm":
        return _product(s["a"].float(), s["b"].float(), s["a_scales"], s["b_scales"], s["bias"], s["type"])
    if kind == "linear":
        q, scale = _quantise(s["x"])
        return _product(q, s["b"].float(), scale[:, 0], s["b_scales"], s["bias"], s["type"])
    if kind == "cache":
        _write(s)
    return _read(s)


def work(case):
    if case["kind"] in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        bias = n * BYTES[case["bias"]] if case["bias"] else 0
        if case["kind"] == "gemm":
            rows, out = m * k + 4 * m, BYTES[case["out"]]
        else:
            rows, out = m * k * BYTES[case["type"]], BYTES[case["type"]]
        return {"bytes": rows + n * k + 4 * n + bias + m * n * out, "flops": 2 * m * n * k}
    lengths = _lengths(case)
    groups = case["parts"] * case["heads"]
    held, given = case["dim"] + 4, case["dim"] * BYTES[case["type"]]
    total = sum(lengths) * groups * (held + given)
    if case["kind"] == "cache":
        new = sum(min(case["new"], v) for v in lengths)
        total += new * (groups * (held + given) + 8)
    return {"bytes": total, "flops": 0}


def exact(case, seed):
    """The definitions in 64 bits: a code is the integer nearest to x / s for the scale s that is kept (the 32-bit
    number nearest to the largest magnitude over 127)."""
    s = prepare(case, seed)

    def values(x):
        x = x.to(torch.float64)
        top = x.abs().max(dim=-1, keepdim=True).values
        kept = top.div(top.new_tensor(127.0)).to(torch.float32).to(torch.float64)
        return torch.round(x / kept).nan_to_num_(nan=0.0), kept

    if case["kind"] in ("gemm", "linear"):
        if case["kind"] == "gemm":
            a, row = s["a"].to(torch.float64), s["a_scales"].to(torch.float64).unsqueeze(1)
        else:
            a, row = values(s["x"])
        out = torch.matmul(a, s["b"].to(torch.float64).transpose(0, 1)).mul_(row).mul_(s["b_scales"].to(torch.float64))
        return out if s["bias"] is None else out.add_(s["bias"].to(torch.float64))
    parts, pages, page, heads, dim = s["codes"].shape
    held = s["codes"].to(torch.float64) * s["scales"].to(torch.float64).unsqueeze(-1)
    held = held.reshape(parts, pages * page, heads, dim)
    if case["kind"] == "cache":
        count = s["slots"].numel() - case["padding"]
        for p, x in enumerate(s["rows"]):
            q, kept = values(x[:count])
            held[p].index_copy_(0, s["slots"][:count], q * kept)
    table, at = s["page_table"].tolist(), []
    for i, v in enumerate(_lengths(case)):
        pos = torch.arange(v)
        at.append(torch.tensor(table[i])[pos // page] * page + pos % page)
    return tuple(held.index_select(1, torch.cat(at).cuda()).unbind(0))
