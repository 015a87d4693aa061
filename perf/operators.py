"""Cases of the operators a 4-bit text encoder and a 4-bit DiT need, for timing and for comparison.

* ``quantize``     MXFP4 quantisation (E2M1 codes, one power-of-two scale per 32 columns) and reading back
* ``linear``       y = Q(x) W^T + bias with W held in 4 bits and x quantised to 4 bits in the call
* ``lora``         the same product with its LoRA side path, forward and backward
* ``attn``         attention with a learned relative position bias by buckets, forward
* ``attn_train``   the same with its backward (dq, dk, dv and the gradient of the bias table)

``run`` computes the plain form (elementary torch operations in fp32, one rounding at the end) unless
``own`` is set, when it calls the framework. ``exact`` gives the same outputs from the definition in float64.
"""

import bisect
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


# ---- cases ----------------------------------------------------------------------------------------------


def _quantize(rows, cols, dt):
    return {"op": "quantize", "rows": rows, "cols": cols, "dt": dt}


def _linear(m, k, n, bias=True):
    return {"op": "linear", "m": m, "k": k, "n": n, "bias": bias}


def _lora(m, k, n, r):
    return {"op": "lora", "m": m, "k": k, "n": n, "r": r}


def _attn(b, h, hk, sq, sk, d, dt, causal=False, mask="none", train=False, buckets=32, max_distance=128):
    return {"op": "attn_train" if train else "attn", "b": b, "h": h, "hk": hk, "sq": sq, "sk": sk, "d": d, "dt": dt,
            "causal": causal, "mask": mask, "buckets": buckets, "max_distance": max_distance}


def listed():
    cases = {
        # one prompt's text embeddings (512 tokens of width 1024) on their way into a 4-bit projection
        "quantize_text": _quantize(512, 1024, "bf16"),
        # an fp32 checkpoint's adaLN weight, the DiT's widest, quantised when the model is loaded
        "quantize_ada_weight": _quantize(18432, 2048, "f32"),
        # the adaLN modulation of one sample: a single conditioning row against the widest weight
        "linear_ada_1": _linear(1, 2048, 18432),
        # the DiT's MLP up-projection at 1024 px (4096 image tokens): sampling without gradients
        "linear_fc1_4096": _linear(4096, 2048, 8192),
        # a short prompt batch through a projection of a width that fills no tile
        "linear_ragged": _linear(231, 1000, 1111),
        # an attention output projection with LoRA rank 16 at 512 px (1024 image tokens): one training step
        "lora_o_1024": _lora(1024, 2048, 2048, 16),
        # a stacked q/k/v projection with three rank-16 LoRAs at 1024 px: one training step
        "lora_qkv_4096": _lora(4096, 2048, 6144, 48),
        # text-encoder layer while a LoRA trains: four padded prompts of up to 512 tokens
        "attn_train_text_512": _attn(4, 16, 16, 512, 512, 64, "bf16", mask="tail", train=True),
        # long captions, no padding, one sample: the largest training case
        "attn_train_4096": _attn(1, 16, 16, 4096, 4096, 64, "bf16", train=True),
        # fp32 numerics check of a causal decoder layer at odd lengths, heads sharing keys and values
        "attn_train_f32_odd": _attn(2, 6, 3, 203, 331, 40, "f32", causal=True, mask="random", train=True),
        # encoding prompts ahead of training, f16, wide heads
        "attn_encode_1024": _attn(8, 16, 16, 1024, 1024, 128, "f16", mask="tail"),
        # one new token against a long cache of a decoder's keys and values
        "attn_decode_8192": _attn(8, 16, 16, 1, 8192, 64, "bf16", causal=True),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    if v > 64 and rng.random() < 0.5:  # half of the larger sizes are multiples of 64, the rest as drawn
        v = v // 64 * 64
    return v if v != 3072 else v + 8


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        for key in ("bytes", "flops"):
            limits[key] = max(limits.get(key, 0), w[key])
    while True:
        op = rng.choice(["quantize", "linear", "lora", "attn", "attn_train", "decode"])
        if op == "quantize":
            case = _quantize(_log_int(rng, 1, 18432), _log_int(rng, 1, 8192), rng.choice(["bf16", "f16", "f32"]))
        elif op == "linear":
            case = _linear(_log_int(rng, 1, 4096), _log_int(rng, 32, 8192), _log_int(rng, 16, 18432), rng.random() < 0.5)
        elif op == "lora":
            case = _lora(_log_int(rng, 64, 4096), _log_int(rng, 128, 8192) // 8 * 8, _log_int(rng, 128, 8192) // 8 * 8,
                         rng.choice([8, 16, 32, 48, 64]))
        else:
            dt = rng.choice(["bf16", "bf16", "f16", "f32"])
            hk = rng.choice([1, 2, 3, 4, 8, 16])
            h = hk * rng.choice([1, 1, 1, 2, 4])
            d = rng.choice([64, 64, 128, 32, 40, 80, 96])
            b = rng.choice([1, 1, 2, 3, 4, 8])
            causal = rng.random() < 0.4
            mask = rng.choice(["none", "tail", "random"])
            buckets, dist = rng.choice([(32, 128), (32, 128), (16, 64), (64, 256)])
            top = 1024 if dt == "f32" else 4096
            if op == "decode":
                sk = _log_int(rng, 1, 8192)
                case = _attn(b, h, hk, rng.choice([1, 1, 1, 2, 5]), sk, d, dt, causal, mask, False, buckets, dist)
            else:
                sq = _log_int(rng, 1, top)
                sk = sq if rng.random() < 0.6 else _log_int(rng, 1, top)
                case = _attn(b, h, hk, sq, sk, d, dt, causal, mask, op == "attn_train", buckets, dist)
            if case["b"] * case["h"] * case["sq"] * case["sk"] > 16 * 4096 * 4096:
                continue
        if any(v == 3072 for v in case.values() if not isinstance(v, bool)):
            continue
        w = work(case)
        if all(w[key] <= limits[key] for key in limits):
            return case


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        size = 4 if case["dt"] == "f32" else 2
        # the input once, codes and scales (17 bytes per 32 values) written and read, the read-back written as bf16
        return {"bytes": n * size + 2 * n * 17 // 32 + 2 * n, "flops": 3 * n}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k * 17 // 32 + 2 * n * case["bias"] + 2 * m * n, "flops": 2 * m * k * n}
    if op == "lora":
        m, k, n, r = case["m"], case["k"], case["n"], case["r"]
        # x, gy, W (both directions), bias, A, B read; y, dx, dA, dB written
        byts = 2 * (2 * m * k + 2 * m * n) + 2 * n * k * 17 // 32 + 2 * n + 4 * r * (k + n)
        return {"bytes": byts, "flops": 4 * m * n * k + 6 * m * r * (k + n)}
    b, h, hk, sq, sk, d = (case[x] for x in ("b", "h", "hk", "sq", "sk", "d"))
    size = 4 if case["dt"] == "f32" else 2
    q_el, kv_el = b * h * sq * d, b * hk * sk * d
    byts = size * (2 * q_el + 2 * kv_el) + (b * sk if case["mask"] != "none" else 0) + 4 * case["buckets"] * h
    pairs = sq * sk
    if case["causal"]:  # keys a query may see, its position counted from the end of the keys
        off = sk - sq
        pairs = sum(min(max(i + off + 1, 0), sk) for i in range(sq))
    flops = 4 * b * h * pairs * d
    if case["op"] == "attn_train":
        byts += size * (2 * q_el + 2 * kv_el) + 4 * case["buckets"] * h  # gradients: dO read, dq, dk, dv written
        flops = flops * 7 // 2
    return {"bytes": byts, "flops": flops}


# ---- inputs ---------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=_device()) * std


def _activation(g, rows, cols):
    # a LayerNorm's output after its affine: unit rows with a few wide channels
    chan = 1.0 + 3.0 * (torch.rand(cols, generator=g, device=_device()) > 0.98)
    return _randn(g, rows, cols) * chan


def _thresholds(nb, max_distance):
    """Distances at which the bucket of a one-sided range of nb buckets goes up: the first nb // 2 distances have
    a bucket each, the others' buckets are spaced by their logarithm up to max_distance."""
    first = nb // 2
    span = nb - first
    return [i for i in range(1, first)] + [
        # smallest n with (n / first)^span >= (max_distance / first)^s, in whole numbers
        bisect.bisect_left(range(first, max_distance), True,
                           key=lambda n: n ** span * first ** s >= max_distance ** s * first ** span) + first
        for s in range(0, span)]


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    dev = _device()
    if op == "quantize":
        dt = _DT[case["dt"]]
        if case["dt"] == "f32":
            x = _randn(g, case["rows"], case["cols"], std=0.02)
        else:
            x = _activation(g, case["rows"], case["cols"])
        return {"x": x.to(dt)}
    if op in ("linear", "lora"):
        m, k, n = case["m"], case["k"], case["n"]
        s = {"x": _activation(g, m, k).bfloat16(), "weight": _randn(g, n, k, std=0.02).bfloat16(), "bias": None}
        if op == "lora" or case["bias"]:
            s["bias"] = _randn(g, n, std=0.02).bfloat16()
        if op == "lora":
            r = case["r"]
            s["a"] = _randn(g, r, k, std=k ** -0.5).bfloat16()
            s["b"] = _randn(g, n, r, std=0.02).bfloat16()
            s["gy"] = _randn(g, m, n, std=0.1).bfloat16()
        return s
    b, h, hk, sq, sk, d = (case[x] for x in ("b", "h", "hk", "sq", "sk", "d"))
    dt = _DT[case["dt"]]
    # projections' outputs [B, S, heads * d] seen as [B, heads, S, d]
    view = lambda n, s: _randn(g, b, s, n * d).to(dt).view(b, s, n, d).transpose(1, 2)  # noqa: E731
    s = {"q": view(h, sq), "k": view(hk, sk), "v": view(hk, sk), "key_mask": None}
    if not case["causal"]:  # an encoder without a score scale carries 1 / sqrt(d) in its query weights
        s["q"] = s["q"] * d ** -0.5
    s["table"] = _randn(g, case["buckets"], h, std=1.0)
    if case["mask"] == "tail":  # padded prompts: the first fills the row, the others end earlier
        lens = torch.randint(1, sk + 1, (b,), generator=g, device=dev)
        lens[0] = sk
        s["key_mask"] = torch.arange(sk, device=dev)[None, :] < lens[:, None]
    elif case["mask"] == "random":  # tokens dropped anywhere; the last sample has none left
        keep = torch.rand(b, sk, generator=g, device=dev) > 0.3
        if b > 1:
            keep[-1] = False
        s["key_mask"] = keep
    if op == "attn_train":
        s["go"] = _randn(g, b, sq, h * d, std=0.1).to(dt).view(b, sq, h, d).transpose(1, 2)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if own:
        import torch_vulkan_b200 as tv
    if "weight" in s:
        weight = s.pop("weight")
        s["w"] = tv.mx4_quantize(weight) if own else _plain_mx4(weight)
    names = {"lora": ("x", "a", "b"), "attn_train": ("q", "k", "v", "table")}.get(case["op"], ())
    for name in names:
        s[name] = s[name].detach().requires_grad_(True)
    if case["op"].startswith("attn"):
        s["args"] = {"max_distance": case["max_distance"], "bidirectional": not case["causal"], "causal": case["causal"],
                     "scale": 1.0 if not case["causal"] else None,
                     "q_offset": case["sk"] - case["sq"] if case["causal"] else 0}
        nb = case["buckets"] // (1 if case["causal"] else 2)
        s["thresholds"] = torch.tensor(_thresholds(nb, case["max_distance"]), device=_device())
    return s


# ---- plain forms ----------------------------------------------------------------------------------------


def _plain_mx4(x):
    """The values an MXFP4 tensor stands for, in fp32. Blocks of 32 columns share the scale
    2^(floor(log2(largest magnitude)) - 2); each element rounds to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times
    it, ties to the even code, and stops at 6."""
    x = x.float()
    rows, cols = x.shape
    pad = -cols % 32
    blocks = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, 32)
    amax = blocks.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(amax).exponent - 3  # frexp's mantissa lies in [0.5, 1)
    exponent = torch.where(amax > 0, exponent.clamp(-127, 127), -127)
    mag = torch.ldexp(blocks.abs(), -exponent).clamp(max=6.0)
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    val = torch.round(mag / step) * step
    return torch.ldexp(torch.copysign(val, blocks), exponent).view(rows, -1)[:, :cols]


def _plain_attention(s):
    case, a = s["case"], s["args"]
    b, h, hk, sq, sk, d = (case[x] for x in ("b", "h", "hk", "sq", "sk", "d"))
    dev = s["q"].device
    scale = a["scale"] if a["scale"] is not None else d ** -0.5
    q = s["q"].detach().float()
    k, v = (s[n].detach().float().repeat_interleave(h // hk, 1) for n in ("k", "v"))
    keep = torch.ones(1, 1, sq, sk, dtype=torch.bool, device=dev)
    rel = torch.arange(sk, device=dev)[None, :] - (torch.arange(sq, device=dev)[:, None] + a["q_offset"])
    if a["causal"]:
        keep = keep & (rel <= 0)
    if s["key_mask"] is not None:
        m = s["key_mask"]
        keep = keep & m[:, None, None, :]
        v = v.masked_fill(~m[:, None, :, None], 0.0)
        k = k.masked_fill(~m[:, None, :, None], 0.0)
    if a["bidirectional"]:
        bucket = torch.bucketize(rel.abs(), s["thresholds"], right=True) + (rel > 0) * (case["buckets"] // 2)
    else:
        bucket = torch.bucketize((-rel).clamp(min=0), s["thresholds"], right=True)
    table = s["table"].detach().float()
    x = torch.matmul(q, k.transpose(-1, -2)) * scale + table[bucket].permute(2, 0, 1)
    x = x.masked_fill(~keep, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = torch.matmul(p, v)
    dt = s["q"].dtype
    if case["op"] == "attn":
        return {"o": o.to(dt)}
    go = s["go"].float()
    dv = torch.matmul(p.transpose(-1, -2), go)
    dp = torch.matmul(go, v.transpose(-1, -2))
    ds = p * (dp - (go * o).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    # rows upside down and each one place further right: a column of the skewed matrix is one relative position
    skew = torch.nn.functional.pad(ds.sum(0).flip(1), (0, sq)).flatten(1)[:, :-sq].view(h, sq, sk + sq - 1).sum(1)
    position = torch.cat([bucket[:, 0].flip(0), bucket[0, 1:]])  # the bucket of each, from the lowest up
    members = position[:, None] == torch.arange(case["buckets"], device=dev)[None, :]
    dtable = torch.matmul(skew, members.float()).t()
    if h != hk:
        dk, dv = (t.view(b, hk, h // hk, sk, d).sum(2) for t in (dk, dv))
    return {"o": o.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt), "dtable": dtable.to(s["table"].dtype)}


def _plain(s):
    op = s["case"]["op"]
    if op == "quantize":
        return {"values": _plain_mx4(s["x"]).bfloat16()}
    if op == "linear":
        y = torch.matmul(_plain_mx4(s["x"]), s["w"].t())
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return {"y": y.bfloat16()}
    if op == "lora":
        x, a, b, gy = (s[n].detach().float() for n in ("x", "a", "b", "gy"))
        hid = torch.matmul(x, a.t())
        y = torch.matmul(_plain_mx4(x), s["w"].t()) + s["bias"].float() + torch.matmul(hid, b.t())
        dhid = torch.matmul(gy, b)
        dx = torch.matmul(gy, s["w"]) + torch.matmul(dhid, a)
        da, db = torch.matmul(dhid.t(), x), torch.matmul(gy.t(), hid)
        return {n: t.bfloat16() for n, t in (("y", y), ("dx", dx), ("da", da), ("db", db))}
    return _plain_attention(s)


# ---- the framework's calls ------------------------------------------------------------------------------


def _framework(s):
    import torch_vulkan_b200 as tv

    op = s["case"]["op"]
    if op == "quantize":
        return {"values": tv.mx4_dequantize(tv.mx4_quantize(s["x"]))}
    if op == "linear":
        return {"y": tv.mx4_linear(s["x"], s["w"], s["bias"])}
    if op == "lora":
        y = tv.mx4_lora_linear(s["x"], s["w"], s["bias"], s["a"], s["b"])
        dx, da, db = torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["gy"])
        return {"y": y.detach(), "dx": dx, "da": da, "db": db}
    o = tv.bucket_bias_attention(s["q"], s["k"], s["v"], s["table"], key_mask=s["key_mask"], **s["args"])
    if op == "attn":
        return {"o": o}
    dq, dk, dv, dtable = torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["table"]), s["go"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------


def _exact_mx4(x):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], 32):
        blk = x[:, c:c + 32].double()
        top = blk.abs().max(dim=1, keepdim=True).values
        # the largest power of two that is no more than the block's largest magnitude, over four
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))
        e = torch.where(torch.pow(2.0, e + 1) <= top, e + 1, torch.where(torch.pow(2.0, e) > top, e - 1, e))
        unit = torch.pow(2.0, torch.clamp(e - 2, -127, 127))
        a = blk.abs() / unit
        hi = torch.searchsorted(grid, a.contiguous()).clamp(max=7)  # first grid value that is no less
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - a, a - grid[lo]
        take_hi = (up < down) | ((up == down) & (hi % 2 == 0)) | (a >= 6.0)
        out[:, c:c + 32] = torch.sign(blk) * torch.where(take_hi, grid[hi], grid[lo]) * unit
    return out


def _exact_attention(case, s):
    b, h, hk, sq, sk, d = (case[x] for x in ("b", "h", "hk", "sq", "sk", "d"))
    causal, dev = case["causal"], s["q"].device
    train = case["op"] == "attn_train"
    scale = d ** -0.5 if causal else 1.0
    nb = case["buckets"] // (1 if causal else 2)
    first, dist = nb // 2, case["max_distance"]

    def bucket_of(rel):
        n, side = (max(-rel, 0), 0) if causal else (abs(rel), nb if rel > 0 else 0)
        if n < first:
            return n + side
        # floor((nb - first) log(n / first) / log(max_distance / first)), whole numbers settling the ties
        span = nb - first
        t = round(span * math.log(n / first) / math.log(dist / first) + 0.5)
        t = min(max(t, 0), span)
        while t > 0 and n ** span * first ** t < dist ** t * first ** span:
            t -= 1
        return min(first + t, nb - 1) + side

    off = sk - sq if causal else 0
    lut = torch.tensor([bucket_of(r) for r in range(-(sq - 1) - off, sk - off)], device=dev)
    i, j = torch.arange(sq, device=dev)[:, None], torch.arange(sk, device=dev)[None, :]
    bucket = lut[j - i + sq - 1]
    out = {n: torch.zeros(b, heads, length, d, dtype=torch.float64, device=dev)
           for n, heads, length in (("o", h, sq), ("dq", h, sq), ("dk", hk, sk), ("dv", hk, sk))}
    dtable = torch.zeros(case["buckets"], h, dtype=torch.float64, device=dev)
    table = s["table"].double()
    for bi in range(b):
        keep = torch.ones(sq, sk, dtype=torch.bool, device=dev)
        if causal:
            keep &= j <= i + off
        if s["key_mask"] is not None:
            keep &= s["key_mask"][bi][None, :]
        some = keep.any(1, keepdim=True)
        for hi in range(h):
            q, k, v = s["q"][bi, hi].double(), s["k"][bi, hi * hk // h].double(), s["v"][bi, hi * hk // h].double()
            logits = torch.where(keep, scale * (q @ k.t()) + table[:, hi][bucket], -math.inf)
            p = torch.where(some, torch.softmax(torch.where(some, logits, 0.0), 1), 0.0)
            out["o"][bi, hi] = p @ v
            if not train:
                continue
            go = s["go"][bi, hi].double()
            ds = p * (go @ v.t() - ((go * out["o"][bi, hi]).sum(1, keepdim=True)))
            out["dq"][bi, hi] = scale * (ds @ k)
            out["dk"][bi, hi * hk // h] += scale * (ds.t() @ q)
            out["dv"][bi, hi * hk // h] += p.t() @ go
            dtable[:, hi] += torch.bincount(bucket.flatten(), weights=ds.flatten(), minlength=case["buckets"])
    return {**out, "dtable": dtable} if train else {"o": out["o"]}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"values": _exact_mx4(s["x"])}
    if op in ("linear", "lora"):
        w = _exact_mx4(s["weight"])
        y = _exact_mx4(s["x"]) @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if op == "linear":
            return {"y": y}
        x, a, b, gy = (s[n].double() for n in ("x", "a", "b", "gy"))
        return {"y": y + (x @ a.t()) @ b.t(), "dx": gy @ w + (gy @ b) @ a, "da": (gy @ b).t() @ x,
                "db": gy.t() @ (x @ a.t())}
    return _exact_attention(case, s)
