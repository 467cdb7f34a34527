"""Operators between the quantized linears of a decode step or a prefill chunk, and their plain forms:

  norm    the residual's addition and the weighted RMS norm behind it        norm.add_rmsnorm
  codes   the same with int8 codes and a scale per row for a W8A8 linear,    norm.add_rmsnorm (codes=, rotate=)
          rotated by a blockwise Hadamard transform where the weights are
  i8      a W8A8 linear on codes, weights packed once                        linear.I8Linear.encode
  rules   penalties of repeated tokens, biases and grammar masks on logits   sampling.LogitRules.encode
  step    codes and the W8A8 linear that reads them                          both

`run` computes the plain form, or where `own` is true calls the framework. In plain form the operators are sequences of
elementary tensor operations in 32 bits. The int8 codes are defined bit for bit: v = r' * w, butterflies a + b, a - b of spans
1, 2, 4, ..., s = max|v| / 127 and rint(v / s), each operation rounded to 32 bits; so both forms give the same codes.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoded token between two sublayers: the smallest call, latency and host time
        {"name": "norm_2048_r1", "kind": "norm", "rows": 1, "d": 2048, "x": "bf16", "r": "f32", "w": "bf16", "out": "bf16", "pad": 0},
        # a ragged batch of a model whose width is no power of two, all in half precision, rows inside wider buffers
        {"name": "norm_2880_r257", "kind": "norm", "rows": 257, "d": 2880, "x": "f16", "r": "f16", "w": "f32", "out": "f16", "pad": 64},
        # a prefill chunk, fp32 residual
        {"name": "norm_4096_r4096", "kind": "norm", "rows": 4096, "d": 4096, "x": "bf16", "r": "f32", "w": "bf16", "out": "bf16", "pad": 0},
        # a decode batch of four whose linears are W8A8, rotated
        {"name": "codes_4096_r4", "kind": "codes", "rows": 4, "d": 4096, "x": "bf16", "r": "f32", "w": "bf16", "rotate": 256, "pad": 0},
        # a prefill chunk of the same
        {"name": "codes_4096_r2048", "kind": "codes", "rows": 2048, "d": 4096, "x": "bf16", "r": "bf16", "w": "bf16", "rotate": 256, "pad": 0},
        # W8A8 linears: one token (the weights' bytes), a decode batch of odd size, a prefill chunk
        {"name": "i8_14336x4096_r1", "kind": "i8", "rows": 1, "n": 14336, "k": 4096, "y": "f32"},
        {"name": "i8_4096x14336_r37", "kind": "i8", "rows": 37, "n": 4096, "k": 14336, "y": "bf16"},
        {"name": "i8_4096x14336_r2048", "kind": "i8", "rows": 2048, "n": 4096, "k": 14336, "y": "bf16"},
        # the sampler's rules on one row of logits with a short history and a grammar
        {"name": "rules_128000_r1", "kind": "rules", "rows": 1, "vocab": 128000, "x": "f32", "history": 700, "bias": 40, "masks": 1, "loose": 0.02},
        # a batch of eight long conversations, one of them under a grammar; an odd vocabulary
        {"name": "rules_151665_r8", "kind": "rules", "rows": 8, "vocab": 151665, "x": "f32", "history": 16384, "bias": 100, "masks": 1, "loose": 0.5},
        # a large batch over a large vocabulary, logits in bf16, a grammar for every fourth row
        {"name": "rules_262144_r64", "kind": "rules", "rows": 64, "vocab": 262144, "x": "bf16", "history": 2048, "bias": 300, "masks": 16, "loose": 0.9},
        # a prefill chunk's norm and the projection behind it
        {"name": "step_4096x4096_r512", "kind": "step", "rows": 512, "n": 4096, "d": 4096, "x": "bf16", "r": "f32", "w": "bf16", "rotate": 256, "y": "bf16", "pad": 0},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of step between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(round(v / step) * step, -(-lo // step) * step), hi // step * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "codes", "codes", "i8", "i8", "i8", "rules", "rules", "rules", "step"])
    types = list(DT)
    if kind in ("norm", "codes"):
        rotate = 0 if kind == "norm" else rng.choice([0, 32, 256])
        d = _log(rng, 256, 16384, max(rotate, 1)) if rng.random() < 0.5 else rng.choice([2048, 2880 if rotate != 256 else 2816, 4096, 5120, 7680, 14336])
        c = {"kind": kind, "rows": _log(rng, 1, (1 << 24) // d), "d": d, "x": rng.choice(types + ["none"]), "r": rng.choice(types), "w": rng.choice(types),
             "pad": rng.choice([0, 0, 32, 7])}
        c.update({"out": rng.choice(types)} if kind == "norm" else {"rotate": rotate})
        return c
    if kind == "i8":
        n, k = _log(rng, 200, 14336, rng.choice([1, 64])), _log(rng, 512, 14336, rng.choice([16, 128]))
        return {"kind": kind, "rows": _log(rng, 1, min(4096, (2048 * 4096 * 14336) // (n * k))), "n": n, "k": k, "y": rng.choice(types)}
    if kind == "step":
        rotate = rng.choice([32, 256])
        d, n = _log(rng, 1024, 8192, rotate), _log(rng, 512, 8192, 64)
        return {"kind": kind, "rows": _log(rng, 1, 1024), "n": n, "d": d, "x": rng.choice(types), "r": rng.choice(types), "w": rng.choice(types), "rotate": rotate,
                "y": rng.choice(types), "pad": rng.choice([0, 32])}
    rows, vocab = _log(rng, 1, 64), _log(rng, 1000, 262144)
    return {"kind": kind, "rows": rows, "vocab": vocab, "x": rng.choice(types), "history": _log(rng, 1, 16384), "bias": rng.choice([0, _log(rng, 1, 300)]),
            "masks": rng.choice([0, 1, rng.randint(1, rows)]), "loose": rng.choice([0.02, 0.1, 0.5, 0.95])}


# ---- what a program holds before the call -----------------------------------------------------------------------------
def _padded(gen, rows, d, pad, dtype, scale=1.0):
    """Rows of d values inside rows of d + pad."""
    return (scale * torch.randn(rows, d + pad, device=gen.device, generator=gen)).to(dtype)[:, :d]


def _norm_inputs(c, gen):
    rows, d, pad = c["rows"], c["d"], c["pad"]
    x = None if c["x"] == "none" else _padded(gen, rows, d, pad, DT[c["x"]])
    # a residual that has grown over the layers, with a few outlier channels
    r = _padded(gen, rows, d, pad, torch.float32, 3.0)
    r[:, torch.randint(0, d, (3,), device=gen.device, generator=gen)] *= 20.0
    r = r.to(DT[c["r"]])
    w = (1.0 + 0.2 * torch.randn(d, device=gen.device, generator=gen)).to(DT[c["w"]])
    return {"kind": c["kind"], "rows": rows, "d": d, "x": x, "r": r, "w": w, "r_out": None if x is None else torch.empty(rows, d + pad, dtype=r.dtype, device=gen.device)[:, :d]}


def _norm(c, gen):
    s = _norm_inputs(c, gen)
    s["out"] = torch.empty(c["rows"], c["d"], dtype=DT[c["out"]], device=gen.device)
    return s


def _code_buffers(c, gen):
    return {"rotate": c["rotate"], "codes": torch.empty(c["rows"], -(-c["d"] // 16) * 16, dtype=torch.int8, device=gen.device)[:, :c["d"]],
            "scales": torch.empty(c["rows"], dtype=torch.float32, device=gen.device)}


def _codes(c, gen):
    # (8 bits stand for values of 8 bits: bfloat16 holds them)
    return {**_norm_inputs(c, gen), **_code_buffers(c, gen), "values": torch.empty(c["rows"], c["d"], dtype=torch.bfloat16, device=gen.device)}


def _weights(gen, n, k):
    w = torch.randn(n, k, device=gen.device, generator=gen)
    s = w.abs().amax(dim=1) / 127
    return torch.round(w / s[:, None]).to(torch.int8), 0.02 * s


def _i8(c, gen):
    rows, n, k = c["rows"], c["n"], c["k"]
    xq, sx = _weights(gen, rows, k)
    w, sw = _weights(gen, n, k)
    return {"kind": "i8", "rows": rows, "xq": xq, "sx": 50 * sx, "w": w, "sw": sw, "y": torch.empty(rows, n, dtype=DT[c["y"]], device=gen.device), "linear": _linear(w, sw)}


def _step(c, gen):
    w, sw = _weights(gen, c["n"], c["d"])
    sw = sw / c["rotate"]
    return {**_norm_inputs(c, gen), **_code_buffers(c, gen), "w8": w, "sw": sw, "y": torch.empty(c["rows"], c["n"], dtype=DT[c["y"]], device=gen.device),
            "linear": _linear(w, sw)}


def _linear(w, sw):
    if own:
        from ingot_b200.linear import I8Linear

        return I8Linear(w, sw)


def _rules(c, gen):
    rows, V, dev = c["rows"], c["vocab"], gen.device
    rand = lambda *n: torch.rand(*n, device=dev, generator=gen)  # noqa: E731
    s = {"kind": "rules", "rows": rows, "x": (3 * torch.randn(rows, V, device=dev, generator=gen)).to(DT[c["x"]]), "out": torch.empty(rows, V, device=dev)}
    # a conversation repeats few tokens often; of different lengths, one of them new
    L = c["history"]
    s["tokens"] = (rand(rows, L) ** 4 * V).to(torch.int32).clamp(max=V - 1)
    s["lens"] = (L * (0.25 + 0.75 * rand(rows))).to(torch.int32)
    s["lens"][rows // 2:rows // 2 + 1] *= int(rows < 3)
    s["prompt_lens"] = (s["lens"] * rand(rows)).to(torch.int32)
    s["repetition"] = torch.where(rand(rows) < 0.7, 1.0 + 0.3 * rand(rows), torch.ones(rows, device=dev))
    s["presence"] = torch.where(rand(rows) < 0.5, rand(rows), torch.zeros(rows, device=dev))
    s["frequency"] = torch.where(rand(rows) < 0.5, 0.2 * rand(rows), torch.zeros(rows, device=dev))
    # a request's biases name different tokens; rows have different numbers of them
    if c["bias"]:
        n = (c["bias"] * rand(rows)).to(torch.int64)
        s["bias_offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), n.cumsum(0)]).to(torch.int32)
        total, j = int(n.sum()), torch.arange(int(n.sum()), device=dev)
        first = torch.randint(0, V, (rows,), device=dev, generator=gen).repeat_interleave(n)
        at = j - s["bias_offsets"][:-1].long().repeat_interleave(n)
        s["bias_tokens"] = ((first + at * (V // (c["bias"] + 1))) % V).to(torch.int32)
        s["bias_values"] = 5 * torch.randn(total, device=dev, generator=gen)
    if c["masks"]:
        words = -(-V // 32)
        allowed = rand(c["masks"], words * 32) < c["loose"]
        if c["masks"] > 2:  # a grammar that has come to its end
            allowed[-1] = False
        bits = allowed.view(c["masks"], words, 32).to(torch.int64) << torch.arange(32, device=dev)
        word = bits.sum(-1)
        s["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
        r = torch.arange(rows, dtype=torch.int32, device=dev)
        every = max(1, rows // c["masks"])
        s["mask_rows"] = torch.where((r % every == 0) & (r // every < c["masks"]), r // every, torch.full_like(r, -1))
    if own:
        from ingot_b200.sampling import LogitRules

        s["rules"] = LogitRules(rows, V, **{n: s.get(n) for n in ("tokens", "prompt_lens", "lens", "repetition", "presence", "frequency", "bias_offsets", "bias_tokens",
                                                                   "bias_values", "mask", "mask_rows")})
    return s


_PREPARE = {"norm": _norm, "codes": _codes, "i8": _i8, "rules": _rules, "step": _step}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return _PREPARE[case["kind"]](case, gen)


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


def _own_norm(s):
    from ingot_b200.norm import add_rmsnorm

    add_rmsnorm(s["x"], s["r"], s["w"], s["rows"], eps=EPS, residual_out=s["r_out"], out=s["out"])
    return {"r": s["r_out"], "out": s["out"]}


def _own_codes(s):
    from ingot_b200.norm import add_rmsnorm

    add_rmsnorm(s["x"], s["r"], s["w"], s["rows"], eps=EPS, residual_out=s["r_out"], codes=s["codes"], scales=s["scales"], rotate=s["rotate"])
    return {"r": s["r_out"], "values": torch.mul(s["codes"], s["scales"][:, None], out=s["values"])}  # what the codes stand for


def _own_i8(s):
    s["linear"].encode(s["xq"], s["sx"], s["y"], s["rows"])
    return s["y"]


def _own_step(s):
    from ingot_b200.norm import add_rmsnorm

    add_rmsnorm(s["x"], s["r"], s["w"], s["rows"], eps=EPS, residual_out=s["r_out"], codes=s["codes"], scales=s["scales"], rotate=s["rotate"])
    s["linear"].encode(s["codes"], s["scales"], s["y"], s["rows"])
    return {"r": s["r_out"], "y": s["y"]}


def _own_rules(s):
    return s["rules"].encode(s["x"], s["rows"], out=s["out"])


def _plain_add(s):
    """(r' as it is stored, its 32-bit values, the weight, 1 / rms)"""
    r = s["r"].float()
    stored = None
    if s["x"] is not None:
        stored = (r + s["x"].float()).to(s["r"].dtype)
        r = stored.float()
    return stored, r, s["w"].float(), torch.rsqrt(r.square().mean(dim=1, keepdim=True) + EPS)


def _plain_norm(s):
    stored, r, w, q = _plain_add(s)
    return {"r": stored, "out": (r * q * w).to(s["out"].dtype)}


def _rotate(v, n):
    """The unnormalised Hadamard transform of every n values of a row, spans 1, 2, 4, ..."""
    rows, d = v.shape
    h = 1
    while h < n:
        p = v.view(rows, d // (2 * h), 2, h)
        v = torch.stack([p[:, :, 0] + p[:, :, 1], p[:, :, 0] - p[:, :, 1]], dim=2).view(rows, d)
        h *= 2
    return v


def _plain_quantize(s):
    stored, r, w, q = _plain_add(s)
    v = _rotate(r * w, s["rotate"])
    step = v.abs().amax(dim=1, keepdim=True) / 127
    return stored, torch.round(v / step), step * q


def _plain_codes(s):
    stored, codes, scales = _plain_quantize(s)
    return {"r": stored, "values": (codes * scales).to(s["values"].dtype)}


def _plain_linear(xq, sx, w, sw, dtype):
    return ((xq.float() @ w.float().T) * sx.view(-1, 1) * sw).to(dtype)


def _plain_i8(s):
    return _plain_linear(s["xq"], s["sx"], s["w"], s["sw"], s["y"].dtype)


def _plain_step(s):
    stored, codes, scales = _plain_quantize(s)
    return {"r": stored, "y": _plain_linear(codes, scales, s["w8"], s["sw"], s["y"].dtype)}


def _plain_rules(s):
    x, dev = s["x"].float(), s["x"].device
    rows, V = x.shape
    at = torch.arange(s["tokens"].shape[1], device=dev)
    prompt, past = at < s["prompt_lens"][:, None], at < s["lens"][:, None]
    # (tokens that do not count go to a column of their own)
    count = lambda which: torch.zeros(rows, V + 1, device=dev).scatter_add_(1, torch.where(which, s["tokens"], V).long(), torch.ones_like(s["tokens"], dtype=torch.float32))[:, :V]  # noqa: E731
    asked, said = count(prompt), count(past & ~prompt)
    rep = s["repetition"][:, None]
    x = torch.where((asked + said) > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * said - s["presence"][:, None] * (said > 0)
    if "bias_values" in s:
        j = torch.arange(s["bias_values"].numel(), device=dev)
        row = torch.searchsorted(s["bias_offsets"][1:].long(), j, right=True)
        x = x.index_put((row, s["bias_tokens"].long()), s["bias_values"], accumulate=True)
    if "mask" in s:
        bits = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=dev)) & 1
        bits = bits.view(s["mask"].shape[0], -1)[:, :V].bool()
        allowed = bits[s["mask_rows"].clamp(min=0).long()] | (s["mask_rows"] < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    return x


_OWN = {"norm": _own_norm, "codes": _own_codes, "i8": _own_i8, "rules": _own_rules, "step": _own_step}
_PLAIN = {"norm": _plain_norm, "codes": _plain_codes, "i8": _plain_i8, "rules": _plain_rules, "step": _plain_step}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    c, kind, rows = case, case["kind"], case["rows"]
    if kind == "i8":
        n, k = c["n"], c["k"]
        return {"bytes": rows * k + n * k + 4 * (rows + n) + rows * n * SIZE[c["y"]], "flops": 2 * rows * n * k}
    if kind == "rules":
        V, words = c["vocab"], -(-c["vocab"] // 32)
        lists = rows * (c["history"] * 0.625 * 4 + 5 * 4 + c["bias"] * 0.5 * 8) + c["masks"] * words * 4
        return {"bytes": rows * V * (SIZE[c["x"]] + 4) + lists, "flops": rows * V}
    d = c["d"]
    moved = d * SIZE[c["w"]] + rows * d * SIZE[c["r"]] + (0 if c["x"] == "none" else rows * d * (SIZE[c["x"]] + SIZE[c["r"]]))
    ops = rows * d * 5
    if kind == "norm":
        return {"bytes": moved + rows * d * SIZE[c["out"]], "flops": ops}
    moved, ops = moved + rows * (d + 4), ops + rows * d * int(math.log2(max(1, c["rotate"])))
    if kind == "step":
        n = c["n"]
        moved, ops = moved + n * d + 4 * n + rows * n * SIZE[c["y"]], ops + 2 * rows * n * d
    return {"bytes": moved, "flops": ops}


# ---- the definitions in 64 bits, on the same inputs -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "i8":
        y = torch.einsum("tk,ok->to", s["xq"].double(), s["w"].double())
        return torch.einsum("to,t,o->to", y, s["sx"].double(), s["sw"].double())
    if s["kind"] == "rules":
        return _exact_rules(s)
    total = s["r"].double()
    if s["x"] is not None:
        total = total + s["x"].double()
    stored = None if s["x"] is None else total
    # what follows goes by the residual as it is stored
    kept = total.float().to(s["r"].dtype).double()
    rms = torch.linalg.vector_norm(kept, dim=1, keepdim=True).square().div(kept.shape[1]).add(EPS).sqrt()
    normed = torch.einsum("td,d->td", kept, s["w"].double()) / rms
    if s["kind"] == "norm":
        return {"r": stored, "out": normed}
    n = max(1, s["rotate"])
    h = torch.ones(1, 1, dtype=torch.float64, device=normed.device)
    while h.shape[0] < n:
        h = torch.kron(torch.tensor([[1.0, 1.0], [1.0, -1.0]], dtype=torch.float64, device=normed.device), h)
    turned = torch.einsum("tbi,ij->tbj", normed.reshape(normed.shape[0], -1, n), h).reshape(normed.shape)
    if s["kind"] == "codes":
        most = turned.abs().max(dim=1, keepdim=True).values
        return {"r": stored, "values": torch.round(turned * 127 / most) * most / 127}
    most = turned.abs().max(dim=1, keepdim=True).values
    y = torch.einsum("tk,ok->to", torch.round(turned * 127 / most), s["w8"].double())
    return {"r": stored, "y": y * (most / 127) * s["sw"].double()}


def _exact_rules(s):
    x = s["x"].double().cpu()
    V = x.shape[1]
    for t in range(x.shape[0]):
        n, p = int(s["lens"][t]), int(s["prompt_lens"][t])
        history = s["tokens"][t, :n].cpu().long()
        said = torch.bincount(history[p:], minlength=V).double()
        seen = torch.bincount(history, minlength=V) > 0
        rep, pres, freq = (float(s[k][t]) for k in ("repetition", "presence", "frequency"))
        row = x[t]
        row[seen] = torch.where(row[seen] > 0, row[seen] / rep, row[seen] * rep)
        row -= freq * said + pres * (said > 0).double()
        if "bias_values" in s:
            a, b = int(s["bias_offsets"][t]), int(s["bias_offsets"][t + 1])
            row[s["bias_tokens"][a:b].cpu().long()] += s["bias_values"][a:b].double().cpu()
        m = int(s["mask_rows"][t]) if "mask" in s else -1
        if m >= 0:
            word = s["mask"][m].cpu().long() & 0xFFFFFFFF
            v = torch.arange(V)
            row[((word[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return x
