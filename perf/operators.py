"""Cases of the microscaled low-bit operators: what is measured of them, and in what form.

Four operators, each measured as a user's program calls it:

  roundtrip  a matrix is quantised to 4-bit microscaled floating point (e2m1 elements, one
             power-of-two scale per 32 of a row) and read back as the values it stands for
  linear     a block linear on a weight held in that form: the rows that come in are quantised
             in the call, then multiplied
  cache      keys and values are quantised into the slots of a paged 8- or 4-bit cache as they
             are written, and read back from other slots
  attend     one query per sequence and head over the cached keys and values of its pages

``own`` picks the side: the plain form below in elementary torch operations, or the
framework's calls.  ``exact`` restates each operator in 64 bits, apart from the plain form.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 32                      # elements that share a scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZEOF = {"bf16": 2, "fp16": 2, "fp32": 4}


def _fk():
    from __graft_entry__ import load_package
    load_package()
    from vdit import fast_kernels
    return fast_kernels


# ------------------------------------------------------------------------------ cases

def listed():
    return [
        # the context vector of the 1-token branch: one row, all latency
        {"name": "roundtrip_token", "op": "roundtrip", "rows": 1, "cols": 1536, "dtype": "bf16"},
        # the SwiGLU output that ffn1 multiplies, 16384 voxels
        {"name": "roundtrip_ffn_rows", "op": "roundtrip", "rows": 16384, "cols": 3840, "dtype": "bf16"},
        # an ffn0 weight as it is loaded, fp32
        {"name": "roundtrip_weight", "op": "roundtrip", "rows": 7680, "cols": 1536, "dtype": "fp32"},
        # ffn0 of the context vector: one row, the weight is all there is to read
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 7680, "k": 1536},
        # an output projection of the 4101 context tokens (64 x 64 patches and 5 more)
        {"name": "linear_context", "op": "linear", "rows": 4101, "n": 1536, "k": 1536},
        # ffn0 of 16384 voxels, the widest linear of a block
        {"name": "linear_ffn0", "op": "linear", "rows": 16384, "n": 7680, "k": 1536},
        # ffn1 of one of the small real samples (4632 voxels), the longest sum
        {"name": "linear_ffn1_small", "op": "linear", "rows": 4632, "n": 1536, "k": 3840},
        # the keys and values of one block's context tokens, 8 bits
        {"name": "cache_context", "op": "cache", "tokens": 4101, "heads": 12, "head_dim": 128, "bits": 8,
         "page": 64},
        # the keys and values of 32768 voxels, 16 x 96 heads, 4 bits
        {"name": "cache_voxels", "op": "cache", "tokens": 32768, "heads": 16, "head_dim": 96, "bits": 4,
         "page": 128},
        # one query over one sample's context: the shortest call that still splits its keys
        {"name": "attend_context", "op": "attend", "batch": 1, "longest": 4101, "heads": 12, "kv_heads": 12,
         "head_dim": 128, "bits": 8, "page": 64},
        # sixteen samples of different lengths, 4 bits, four queries sharing each key head
        {"name": "attend_ragged", "op": "attend", "batch": 16, "longest": 6082, "heads": 16, "kv_heads": 4,
         "head_dim": 96, "bits": 4, "page": 16},
        # sixteen samples of up to 32768 voxels, 8 bits: reading the cache is all the time
        {"name": "attend_voxels", "op": "attend", "batch": 16, "longest": 32768, "heads": 12, "kv_heads": 12,
         "head_dim": 128, "bits": 8, "page": 128},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["roundtrip", "linear", "linear", "cache", "attend", "attend"])
    if op == "roundtrip":
        cols = BLOCK * _spread(rng, 1, 240)
        return {"op": op, "rows": _spread(rng, 1, min(32768, 62_000_000 // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "linear":
        k = BLOCK * _spread(rng, 2, 120)
        n = 8 * _spread(rng, 4, 960)
        return {"op": op, "rows": _spread(rng, 1, min(32768, 190_000_000_000 // (n * k))), "n": n, "k": k}
    head_dim, heads = rng.choice([(32, 6), (64, 8), (96, 16), (96, 5), (128, 12), (128, 3)])
    bits, page = rng.choice([8, 8, 4]), rng.choice([16, 32, 64, 128])
    if op == "cache":
        return {"op": op, "tokens": _spread(rng, 1, 32768), "heads": heads, "head_dim": head_dim, "bits": bits,
                "page": page}
    return {"op": op, "batch": _spread(rng, 1, 16), "longest": _spread(rng, 1, 32768),
            "heads": heads * rng.choice([1, 1, 2, 4]), "kv_heads": heads, "head_dim": head_dim, "bits": bits,
            "page": page}


def _lengths(case):
    """The sequences' lengths: the longest first, the others a quarter of it to all of it, and
    in a batch of three or more one sequence that holds nothing yet."""
    rng = random.Random(case["batch"] * 1_000_003 + case["longest"])
    out = [case["longest"]] + [int(case["longest"] * rng.uniform(0.25, 1.0)) for _ in range(case["batch"] - 1)]
    if len(out) >= 3:
        out[len(out) // 2] = 0
    return out


def work(case):
    op = case["op"]
    if op == "roundtrip":
        n = case["rows"] * case["cols"]
        held = n // 2 + n // BLOCK
        return {"bytes": n * SIZEOF[case["dtype"]] * 2 + 2 * held, "flops": 0}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k * 2 + n * k // 2 + n * k // BLOCK + n * 2 + m * n * 2, "flops": 2 * m * n * k}
    width = case["head_dim"] * case["bits"] // 8 + case["head_dim"] // BLOCK     # bytes of a key of one head
    if op == "cache":
        t, d = case["tokens"], case["heads"] * case["head_dim"]
        return {"bytes": t * 8 + 2 * t * d * 2 + 2 * t * case["heads"] * width * 2 + 2 * t * d * 2, "flops": 0}
    keys = sum(_lengths(case))
    d = case["heads"] * case["head_dim"]
    return {"bytes": keys * case["kv_heads"] * width * 2 + case["batch"] * d * 4, "flops": 4 * keys * d}


# ------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _rows(g, rows, cols, dtype):
    """Modulated rows: unit normal, channels of different gain, a few of them large."""
    gain = torch.rand(cols, generator=g, device=DEVICE) + 0.5
    gain = torch.where(torch.rand(cols, generator=g, device=DEVICE) < 0.01, gain * 12, gain)
    return (torch.randn(rows, cols, generator=g, device=DEVICE) * gain).to(dtype)


def _inputs(case, seed):
    """The operator's arguments, before anything is quantised."""
    g, op = _gen(seed), case["op"]
    if op == "roundtrip":
        return {"x": _rows(g, case["rows"], case["cols"], DTYPES[case["dtype"]])}
    if op == "linear":
        n, k = case["n"], case["k"]
        return {"x": _rows(g, case["rows"], k, torch.bfloat16),
                "w": (torch.randn(n, k, generator=g, device=DEVICE) * 0.02).to(torch.bfloat16),
                "bias": (torch.randn(n, generator=g, device=DEVICE) * 0.02).to(torch.bfloat16)}
    page, d = case["page"], case["head_dim"]
    if op == "cache":
        t, h = case["tokens"], case["heads"]
        pages = -(-t // page) + 1
        slots = torch.randperm(pages * page, generator=g, device=DEVICE)[:t]
        return {"k": _rows(g, t, h * d, torch.bfloat16), "v": _rows(g, t, h * d, torch.bfloat16), "slots": slots,
                "back": slots[torch.randperm(t, generator=g, device=DEVICE)], "pages": pages}
    lengths, h = _lengths(case), case["kv_heads"]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    # normalised queries and keys, as behind a QK norm
    return {"q": torch.randn(case["batch"], case["heads"] * d, generator=g, device=DEVICE).to(torch.bfloat16),
            "k": torch.randn(pages * page, h * d, generator=g, device=DEVICE).to(torch.bfloat16),
            "v": torch.randn(pages * page, h * d, generator=g, device=DEVICE).to(torch.bfloat16),
            "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE), "pages": pages,
            "host_lengths": lengths}


# ------------------------------------------------------------------------------ plain form

def _plain_quantise(x, bits):
    """(elements, exponents) of rows x [R, C]: elements on the e2m1 or e4m3 grid, held as
    float8 e4m3 (which has every e2m1 value), and one int8 exponent per 32."""
    b = x.to(torch.float32).reshape(x.shape[0], -1, BLOCK)
    top, grid_max, mant, low = (2, 6.0, 1, 0) if bits == 4 else (8, 448.0, 3, -6)
    e = (torch.frexp(b.abs().amax(-1)).exponent - 1 - top).clamp_(min=-127)
    y = torch.ldexp(b, -e.unsqueeze(-1))
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp_(min=low) - mant)
    y = (torch.round(y / step) * step).clamp_(-grid_max, grid_max)
    return y.to(torch.float8_e4m3fn).reshape(x.shape), e.to(torch.int8)


def _plain_values(elements, exponents):
    b = elements.to(torch.float32).reshape(*exponents.shape, BLOCK)
    return torch.ldexp(b, exponents.to(torch.int32).unsqueeze(-1)).reshape(elements.shape)


def prepare(case, seed):
    s, op = _inputs(case, seed), case["op"]
    s["case"] = case
    fk = _fk() if own else None
    if op == "linear":
        w = s.pop("w")
        s["w"] = fk.quantize_mxfp4(w) if own else _plain_quantise(w, 4)
    elif op in ("cache", "attend"):
        h = case["kv_heads"] if op == "attend" else case["heads"]
        rows = s["pages"] * case["page"]
        if own:
            s["cache"] = fk.MxKvCache(s["pages"], case["page"], h, case["head_dim"], bits=case["bits"],
                                      device=DEVICE)
        if op == "attend":
            k, v = s.pop("k"), s.pop("v")
            if own:
                fk.kv_cache_write(s["cache"], k, v, torch.arange(rows, device=DEVICE))
            else:
                s["k"], s["v"] = _plain_quantise(k, case["bits"]), _plain_quantise(v, case["bits"])
        elif not own:
            d = h * case["head_dim"]
            s["cache"] = [(torch.zeros(rows, d, device=DEVICE, dtype=torch.float8_e4m3fn),
                           torch.zeros(rows, d // BLOCK, device=DEVICE, dtype=torch.int8)) for _ in range(2)]
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    fk, case = _fk(), s["case"]
    op = case["op"]
    if op == "roundtrip":
        return fk.dequantize_mxfp4(fk.quantize_mxfp4(s["x"]), s["x"].dtype)
    if op == "linear":
        return fk.linear_mxfp4(s["x"], s["w"], s["bias"])
    if op == "cache":
        fk.kv_cache_write(s["cache"], s["k"], s["v"], s["slots"])
        return fk.kv_cache_read(s["cache"], s["back"])
    return fk.attention_1q_cached(s["q"], s["cache"], s["table"], s["lengths"])


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "roundtrip":
        return _plain_values(*_plain_quantise(s["x"], 4)).to(s["x"].dtype)
    if op == "linear":
        x = _plain_values(*_plain_quantise(s["x"], 4))
        return (x @ _plain_values(*s["w"]).t() + s["bias"].to(torch.float32)).to(torch.bfloat16)
    if op == "cache":
        out = []
        for rows, (elements, exponents) in zip((s["k"], s["v"]), s["cache"]):
            y, e = _plain_quantise(rows, case["bits"])
            elements[s["slots"]], exponents[s["slots"]] = y, e
            out.append(_plain_values(elements[s["back"]], exponents[s["back"]]).to(torch.bfloat16))
        return tuple(out)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    q = s["q"].to(torch.float32).reshape(case["batch"], hk, h // hk, d) / math.sqrt(d)
    out = torch.zeros(case["batch"], hk, h // hk, d, device=DEVICE)
    step = torch.arange(case["page"], device=DEVICE)
    for i, n in enumerate(s["host_lengths"]):
        if n == 0:
            continue                                        # nothing to attend to: zeros
        pages = s["table"][i, :-(-n // case["page"])].to(torch.int64)
        rows = (pages.unsqueeze(1) * case["page"] + step).reshape(-1)[:n]
        k, v = (_plain_values(t[0][rows], t[1][rows]).reshape(n, hk, d) for t in (s["k"], s["v"]))
        a = torch.softmax(torch.einsum("hgd,nhd->hgn", q[i], k), -1)
        out[i] = torch.einsum("hgn,nhd->hgd", a, v)
    return out.reshape(case["batch"], h * d).to(torch.bfloat16)


# ------------------------------------------------------------------------------ 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _two_to(e):
    """2^e in 64 bits, exactly (torch.pow is off by an ulp for some whole exponents)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_values(x, bits):
    """What rows x stand for once held in ``bits``, from the format's definition in 64 bits:
    the block's exponent is that of its largest magnitude less the element type's own, each
    element goes to the nearest value of its type, halves to the even one, and no further than
    the largest."""
    b = x.to(torch.float64).reshape(x.shape[0], -1, BLOCK)
    big = b.abs().amax(-1, keepdim=True)
    exponent = torch.floor(torch.log2(torch.where(big > 0, big, torch.ones_like(big))))
    # log2 next to a power of two may round to the other side of it
    exponent = torch.where(_two_to(exponent) > big, exponent - 1, exponent)
    exponent = torch.where(_two_to(exponent + 1) <= big, exponent + 1, exponent)
    unit = _two_to(torch.where(big > 0, exponent - (2 if bits == 4 else 8), torch.full_like(big, -127)).clamp(min=-127))
    y = (b / unit).abs()
    if bits == 4:
        grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
        middle = (grid[1:] + grid[:-1]) / 2
        i = torch.bucketize(y, middle)                      # a value on a middle goes to the lower index ...
        on = (i < 7) & (y == middle[i.clamp(max=6)])
        i = torch.where(on & (i % 2 == 1), i + 1, i)        # ... unless that is the odd one
        y = grid[i]
    else:
        unit_y = torch.full_like(y, 2.0 ** -9)              # subnormals and the first binade
        for p in range(-5, 9):
            unit_y = torch.where(y >= 2.0 ** p, torch.full_like(y, 2.0 ** (p - 3)), unit_y)
        y = (torch.round(y / unit_y) * unit_y).clamp(max=448.0)
    return (torch.copysign(y, b) * unit).reshape(x.shape)


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "roundtrip":
        return _exact_values(s["x"], 4)
    if op == "linear":
        w = _exact_values(s["w"], 4)
        parts = [_exact_values(p, 4) @ w.t() + s["bias"].to(torch.float64) for p in s["x"].split(4096)]
        return torch.cat(parts)
    if op == "cache":
        place = torch.empty(s["pages"] * case["page"], dtype=torch.int64, device=DEVICE)
        place[s["slots"]] = torch.arange(case["tokens"], device=DEVICE)
        return tuple(_exact_values(s[n], case["bits"])[place[s["back"]]] for n in ("k", "v"))
    hk, d, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // hk
    out = torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(s["host_lengths"]):
        if n == 0:
            continue
        at = torch.arange(n, device=DEVICE)
        rows = s["table"][i].to(torch.int64)[at // page] * page + at % page
        k = _exact_values(s["k"][rows], case["bits"]).reshape(n, hk, d)
        v = _exact_values(s["v"][rows], case["bits"]).reshape(n, hk, d)
        q = s["q"][i].to(torch.float64).reshape(case["heads"], d)
        for j in range(case["heads"]):
            score = (k[:, j // group] @ q[j]) / math.sqrt(d)
            p = torch.exp(score - score.max())
            out[i, j] = (p @ v[:, j // group]) / p.sum()
    return out.reshape(case["batch"], -1)
