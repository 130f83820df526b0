"""Measured cases of the 8-bit product and the attention operators.

Three operators, the arithmetic of one attention block of a quantised
speech encoder or decoder:

  quantize_rows  symmetric 8-bit values and one scale for each row (token);
  matmul_int8    int8 x int8 product with a scale for each token and each
                 output channel, an optional bias, float32 or float16 result;
  attention      softmax(q k^T * scale) v of queries over keys and values of
                 another length, with key lengths and a key mask.

``run`` computes a case in plain float32 torch operations, or, where ``own``
is true, by the calls of ``bt_b200.runtime.BtRuntime``.
"""
import functools
import math
import os
import sys

import torch

own = False


# ---- the cases ----------------------------------------------------------------
def _quant(name, rows, k, dtype):
    return {"name": name, "op": "quantize_rows", "rows": rows, "k": k, "dtype": dtype}


def _matmul(name, m, n, k, out, bias):
    return {"name": name, "op": "matmul_int8", "m": m, "n": n, "k": k, "out": out, "bias": bias}


def _attn(name, b, h, hkv, tq, tk, d, dtype, keys, layout):
    return {"name": name, "op": "attention", "b": b, "h": h, "hkv": hkv, "tq": tq, "tk": tk, "d": d, "dtype": dtype,
            "keys": keys, "layout": layout}


def listed():
    return [
        # one token's hidden state before a quantised projection: latency
        _quant("quantize one token", 1, 768, "float32"),
        # the feed-forward activations of a batch of 64 utterances of 510 tokens
        _quant("quantize batch", 32640, 2048, "float32"),
        # one token through the feed-forward's first projection: latency
        _matmul("matmul one token", 1, 2048, 768, "float32", True),
        # one utterance through the feed-forward's second projection
        _matmul("matmul utterance", 510, 768, 2048, "float32", True),
        # a batch of 64 utterances through the first projection
        _matmul("matmul batch", 32640, 2048, 768, "float16", True),
        # a few tokens by odd sizes: a vocabulary-like output, no bias
        _matmul("matmul ragged", 77, 5001, 1000, "float32", False),
        # a wide model's projection over a long prompt
        _matmul("matmul wide", 16384, 8192, 8192, "float16", False),
        # the text encoder's attention over a padded batch of 64 utterances
        _attn("attention text batch", 64, 12, 12, 510, 510, 64, "float16", "lengths", "token"),
        # audio frames attending to the text encoder's states, masked keys
        _attn("attention frames to text", 16, 16, 16, 1500, 333, 64, "float16", "mask", "token"),
        # long audio attending to a longer context, shared key heads
        _attn("attention long", 1, 16, 4, 4096, 16384, 128, "float16", "all", "head"),
        # one decoding step of 32 sequences over their encoder states
        _attn("attention one token", 32, 16, 16, 1, 2000, 64, "float16", "lengths", "head"),
        # the float32 model as it stands, 8 utterances
        _attn("attention float32", 8, 12, 12, 510, 510, 64, "float32", "lengths", "token"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize_rows", "matmul_int8", "matmul_int8", "attention", "attention", "attention"])
    while True:
        if op == "quantize_rows":
            c = _quant("", _log(rng, 1, 40000), _log(rng, 16, 16384), rng.choice(["float32", "float16"]))
            if c["rows"] * c["k"] <= 1 << 27:
                break
        elif op == "matmul_int8":
            c = _matmul("", _log(rng, 1, 33000), _log(rng, 64, 16384), _log(rng, 64, 16384),
                        rng.choice(["float32", "float16"]), rng.choice([True, False]))
            if c["m"] * c["n"] * c["k"] <= 1 << 40 and c["m"] * c["n"] <= 1 << 28:
                break
        else:
            hkv = rng.choice([1, 2, 4, 8, 12, 16])
            h = hkv * rng.choice([1, 1, 1, 2, 4, 8])
            tq = 1 if rng.random() < 0.3 else _log(rng, 2, 6000)
            c = _attn("", _log(rng, 1, 64), h, hkv, tq, _log(rng, 1, 20000), rng.choice([32, 40, 64, 64, 80, 96, 128, 128]),
                      rng.choice(["float16", "float16", "float16", "float32"]), rng.choice(["all", "lengths", "mask"]),
                      rng.choice(["token", "head"]))
            scores = c["b"] * c["h"] * c["tq"] * c["tk"]
            states = c["b"] * c["d"] * (c["h"] * c["tq"] + c["hkv"] * c["tk"])
            if scores <= (1 << 30 if c["dtype"] == "float16" else 1 << 26) and states <= 1 << 28:
                break
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------
def _lengths(c):
    """Key lengths of a padded batch: spread from half of tk to tk."""
    if c["b"] == 1:
        return [c["tk"]]
    return [max(1, c["tk"] - (c["tk"] // 2) * i // (c["b"] - 1)) for i in range(c["b"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = case

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"op": c["op"]}
    if c["op"] == "quantize_rows":
        # activations with a few louder channels, as hidden states have
        gain = torch.exp(0.5 * randn(c["k"]))
        s["x"] = (randn(c["rows"], c["k"]) * gain).to(getattr(torch, c["dtype"]))
    elif c["op"] == "matmul_int8":
        def codes(rows):
            v = (randn(rows, (c["k"] + 15) // 16 * 16) * 36).round_().clamp_(-127, 127).to(torch.int8)
            return v[:, :c["k"]]   # rows on 16-byte boundaries, as quantize_rows lays them out
        s["a"], s["w"] = codes(c["m"]), codes(c["n"])
        s["a_scale"] = 0.01 + 0.02 * torch.rand(c["m"], generator=g, device="cuda")
        s["w_scale"] = 1e-4 + 1e-3 * torch.rand(c["n"], generator=g, device="cuda")
        s["bias"] = randn(c["n"]) if c["bias"] else None
        s["out"] = getattr(torch, c["out"])
    else:
        dt = getattr(torch, c["dtype"])

        def states(heads, length):
            if c["layout"] == "token":
                return randn(c["b"], length, heads, c["d"]).to(dt).permute(0, 2, 1, 3)
            return randn(c["b"], heads, length, c["d"]).to(dt)
        s["q"], s["k"], s["v"] = states(c["h"], c["tq"]), states(c["hkv"], c["tk"]), states(c["hkv"], c["tk"])
        s["lengths"] = s["mask"] = None
        if c["keys"] == "lengths":
            order = torch.randperm(c["b"], generator=g, device="cuda")
            s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")[order].contiguous()
        elif c["keys"] == "mask":
            s["mask"] = torch.rand((c["b"], c["tk"]), generator=g, device="cuda") < 0.9
    return s


# ---- one pass -----------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _runtime():
    path = os.path.join(os.getcwd(), "best-tts-godot_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from bt_b200.runtime import BtRuntime
    return BtRuntime(0)


def _plain_quantize_rows(x):
    x = x.float()
    top = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    q = torch.round(x * (torch.full_like(top, 127.0) / top))
    return q.nan_to_num(nan=0.0).to(torch.int8), (top / torch.full_like(top, 127.0)).squeeze(-1)


def _plain_matmul_int8(a, a_scale, w, w_scale, bias, out):
    y = (a.float() @ w.float().t()) * (a_scale[:, None] * w_scale)
    return (y if bias is None else y + bias).to(out)


def _plain_attention(q, k, v, lengths, mask):
    b, h, tq, d = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    s = q.float().reshape(b, hkv, h // hkv * tq, d) @ k.float().transpose(-1, -2)
    s *= 1.0 / math.sqrt(d)
    if lengths is not None:
        mask = torch.arange(tk, device=q.device) < lengths[:, None]
    v = v.float()
    if mask is not None:
        s.masked_fill_(~mask[:, None, None, :], -math.inf)
        v = v.masked_fill(~mask[:, None, :, None], 0.0)
    s = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    o = (s @ v) / s.sum(-1, keepdim=True).clamp_min(1e-37)
    return o.reshape(b, h, tq, d).to(q.dtype)


def run(state):
    s = state
    if own:
        rt = _runtime()
        if s["op"] == "quantize_rows":
            return rt.quantize_rows(s["x"])
        if s["op"] == "matmul_int8":
            return rt.matmul_int8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], out_dtype=s["out"])
        return rt.attention(s["q"], s["k"], s["v"], lengths=s["lengths"], key_mask=s["mask"])
    if s["op"] == "quantize_rows":
        return _plain_quantize_rows(s["x"])
    if s["op"] == "matmul_int8":
        return _plain_matmul_int8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["out"])
    return _plain_attention(s["q"], s["k"], s["v"], s["lengths"], s["mask"])


# ---- what a pass cannot do without --------------------------------------------
def _size(dtype):
    return {"float32": 4, "float16": 2}[dtype]


def work(case):
    c = case
    if c["op"] == "quantize_rows":
        n = c["rows"] * c["k"]
        return {"bytes": n * (_size(c["dtype"]) + 1) + 4 * c["rows"], "flops": 2 * n}
    if c["op"] == "matmul_int8":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + 4 * m + 4 * n * (2 if c["bias"] else 1) + m * n * _size(c["out"]),
                "flops": 2 * m * n * k}
    keys = sum(_lengths(c)) if c["keys"] == "lengths" else c["b"] * c["tk"]
    item = _size(c["dtype"])
    tail = 4 * c["b"] if c["keys"] == "lengths" else c["b"] * c["tk"] if c["keys"] == "mask" else 0
    return {"bytes": 2 * item * c["b"] * c["h"] * c["tq"] * c["d"] + 2 * item * c["hkv"] * keys * c["d"] + tail,
            "flops": 4 * c["h"] * c["tq"] * keys * c["d"]}


# ---- the definitions in 64 bits ------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize_rows":
        x = s["x"].double()
        largest = torch.maximum(x.max(dim=-1).values, -x.min(dim=-1).values)
        largest = torch.clamp(largest, min=2.0 ** -100)
        return None, largest / 127.0   # the codes are whole numbers of float32 products
    if s["op"] == "matmul_int8":
        y = torch.einsum("mk,nk->mn", s["a"].double(), s["w"].double())
        y = y.mul_(s["a_scale"].double().unsqueeze(1)).mul_(s["w_scale"].double().unsqueeze(0))
        return y if s["bias"] is None else y.add_(s["bias"].double())
    q, k, v = s["q"], s["k"], s["v"]
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(q.shape[0]):
        kept = torch.arange(k.shape[2], device=q.device)
        if s["lengths"] is not None:
            kept = kept[: int(s["lengths"][i])]
        if s["mask"] is not None:
            kept = kept[s["mask"][i]]
        if kept.numel() == 0:
            continue
        for j in range(k.shape[1]):
            kk, vv = k[i, j].double()[kept], v[i, j].double()[kept]
            for n in range(j * group, (j + 1) * group):
                out[i, n] = torch.softmax(torch.einsum("td,sd->ts", q[i, n].double(), kk) / math.sqrt(q.shape[3]), -1) @ vv
    return out
