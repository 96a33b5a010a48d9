"""The 8-bit operators of the sampling path, as they are timed and compared with their plain forms.

The storage format is the same throughout: e4m3 values in blocks of 128 consecutive elements of the last axis, one
power-of-two scale (e8m0) a block. With amax the largest magnitude of a block, the scale is the least power of two
with amax <= 448 * scale and the codes are x / scale rounded to nearest even. The scales of a matrix [rows, cols]
are held as [ceil(blocks / 4), rows, 4] (four blocks of a row in one 32-bit word, zero bytes behind the last block);
those of a cache as [batch, layers, 2, heads, capacity].

  quantize   a matrix to that format (activations row by row; weights are the same call, made once)
  adaln      RMS norm, scale and shift of the residual stream, quantised as it is written
  gemm       the product of two such matrices, with the tails of the decoder's projections
  kv_write   keys (head norm and rotary positions on the way) and values of all layers quantised into a cache
  attention  bf16 queries over bf16 keys of their own sequence and the quantised caches, gated
"""
import math

import torch

own = False

BLOCK = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
PART = 0.5625  # what _lengths draws of a capacity, on average


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # activations of one blockwise step, in fp32, with a last block that is cut short
        {"name": "quantize 157x1360 fp32", "op": "quantize", "rows": 157, "cols": 1360, "type": "fp32", "gap": 0},
        # the attention output of a batch of 16 prompts under two guidances (48 rows of 640 latents)
        {"name": "quantize 30720x2048", "op": "quantize", "rows": 30720, "cols": 2048, "type": "bf16", "gap": 0},
        # the residual stream of one prompt; the same of the batch of 16 under two guidances
        {"name": "adaln 640x2048", "op": "adaln", "rows": 640, "dim": 2048, "vecs": 1, "type": "bf16"},
        {"name": "adaln 30720x2048", "op": "adaln", "rows": 30720, "dim": 2048, "vecs": 1, "type": "bf16"},
        # the closing projection of the MLP in a blockwise step of one prompt: weights are read for few rows
        {"name": "gemm 157x2048x5888 residual", "op": "gemm", "m": 157, "n": 2048, "k": 5888, "tail": "residual", "bias": False},
        # the q, k, v and gate projection of the batch; the gated MLP projection whose output stays in 8 bits
        {"name": "gemm 30720x8192x2048", "op": "gemm", "m": 30720, "n": 8192, "k": 2048, "tail": "store", "bias": False},
        {"name": "gemm 30720x11776x2048 swiglu fp8", "op": "gemm", "m": 30720, "n": 11776, "k": 2048, "tail": "swiglu_fp8", "bias": False},
        # one more token of the latent prefix, all layers; the caches of two speakers' prompts, one of them shorter
        {"name": "kv_write 4x1", "op": "kv_write", "batch": 4, "tokens": 1, "capacity": 160, "layers": 24, "heads": 16, "norm": True,
         "rope": 8, "type": "bf16"},
        {"name": "kv_write 2x1600", "op": "kv_write", "batch": 2, "tokens": 1600, "capacity": 1600, "layers": 24, "heads": 16,
         "norm": True, "rope": 0, "type": "bf16"},
        # one query over text and speaker caches; one prompt, and 16 prompts, under two guidances
        {"name": "attention 16x1", "op": "attention", "prompts": 16, "groups": 1, "queries": 1, "heads": 16, "self": False,
         "text": 768, "speaker": 1600, "gate": False},
        {"name": "attention 3x640", "op": "attention", "prompts": 1, "groups": 3, "queries": 640, "heads": 16, "self": True,
         "text": 768, "speaker": 1600, "gate": True},
        {"name": "attention 48x640", "op": "attention", "prompts": 16, "groups": 3, "queries": 640, "heads": 16, "self": True,
         "text": 768, "speaker": 1600, "gate": True},
    ]


def draw(rng):
    def size(lo, hi, step=1):
        """A multiple of `step` between lo and hi, spread over its logarithm."""
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(step, min(hi // step * step, int(round(v / step)) * step))

    op = rng.choice(["quantize", "adaln", "gemm", "gemm", "kv_write", "attention", "attention"])
    while True:
        if op == "quantize":
            c = {"op": op, "rows": size(1, 30720), "cols": size(16, 5888, 16), "type": rng.choice(["bf16", "fp32"]),
                 "gap": rng.choice([0, 8, 64])}
        elif op == "adaln":
            vecs = rng.choice([1, 1, 3])
            c = {"op": op, "rows": size(1, 10240) * vecs, "dim": rng.choice([size(16, 4096, 16), 1024, 2048]), "vecs": vecs,
                 "type": rng.choice(["bf16", "bf16", "fp32"])}
        elif op == "gemm":
            tail = rng.choice(["store", "residual", "swiglu", "swiglu_fp8"])
            c = {"op": op, "m": size(1, 30720), "n": size(32, 11776, 32), "k": size(64, 5888, 16), "tail": tail,
                 "bias": tail in ("store", "residual") and rng.random() < 0.5}
        elif op == "kv_write":
            heads = rng.choice([1, 2, 10, 16])
            tokens = rng.choice([1, size(2, 1600)])
            c = {"op": op, "batch": size(1, 16), "tokens": tokens, "capacity": tokens + rng.choice([0, 3, 61]), "layers": size(1, 24),
                 "heads": heads, "norm": rng.random() < 0.7, "rope": rng.choice([0, heads // 2, heads]), "type": rng.choice(["bf16", "bf16", "fp32"])}
        else:
            alone = rng.random() < 0.4
            c = {"op": op, "prompts": size(1, 16), "groups": rng.choice([1, 3]), "queries": 1 if alone else size(2, 640),
                 "heads": rng.choice([1, 2, 10, 16]), "self": not alone and rng.random() < 0.8, "text": size(1, 768),
                 "speaker": rng.choice([0, size(1, 1600)]), "gate": rng.random() < 0.5}
        w, top = work(c), max((work(x) for x in listed() if x["op"] == op), key=lambda x: x["bytes"] + x["flops"])
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return c


def work(case):
    c = case
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (_bytes(c) + 1) + n // BLOCK, "flops": 3 * n}
    if c["op"] == "adaln":
        n = c["rows"] * c["dim"]
        return {"bytes": n * (_bytes(c) + 1) + n // BLOCK + 2 * c["vecs"] * c["dim"] * _bytes(c), "flops": 7 * n}
    if c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        read = (m + n) * (k + k // BLOCK)
        out = {"store": 2 * m * n, "residual": 4 * m * n, "swiglu": m * n, "swiglu_fp8": m * n // 2 + m * n // 256}[c["tail"]]
        return {"bytes": read + out, "flops": 2 * m * n * k}
    if c["op"] == "kv_write":
        n = int(c["batch"] * c["tokens"] * c["layers"] * 2 * c["heads"] * 128 * (1 if c["tokens"] == 1 else PART))
        return {"bytes": n * (_bytes(c) + 1) + n // BLOCK, "flops": 5 * n}
    rows, hd = c["prompts"] * c["groups"], c["heads"] * 128
    keys = c["text"] + c["speaker"]
    cached = c["prompts"] * keys * hd * 2 + c["prompts"] * keys * c["heads"] * 2
    io = rows * c["queries"] * hd * 2 * (2 + (2 if c["self"] else 0) + (1 if c["gate"] else 0))
    # a third of the guided rows is without text, a third without speaker
    seen = (c["queries"] if c["self"] else 0) + keys * PART * (2 / 3 if c["groups"] == 3 else 1)
    return {"bytes": cached * PART + io, "flops": 4 * rows * c["queries"] * seen * hd}


def _bytes(c):
    return TYPES[c["type"]].itemsize


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed, device="cuda"):
    g = torch.Generator(device)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, type=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(type)


def _activations(g, rows, cols, type):
    """Rows of differing size with a few loud channels, as behind a norm or an attention."""
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.float32)
    x *= torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))
    return (x * (1 + 20 * (torch.rand((1, cols), generator=g, device="cuda") > 0.99))).to(type)


def _matrix(x):
    """A matrix in the 8-bit format: what a program holds of its weights, or has from the call before."""
    q, e = _quantized(x.float())
    return q.to(E4M3), _words(e)


def _rope(positions):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return torch.stack([angle.cos(), angle.sin()], -1).float().cuda()


def _lengths(g, n, most):
    return torch.randint(max(1, most // 8), most + 1, (n,), generator=g, dtype=torch.int32) if most else torch.zeros(n, dtype=torch.int32)


def prepare(case, seed):
    c, g = case, _generator(seed)
    h = _generator(seed + 1, "cpu")
    s = {"case": c}
    if c["op"] == "quantize":
        s["x"] = _activations(g, c["rows"], c["cols"] + c["gap"], TYPES[c["type"]])[:, :c["cols"]]
    elif c["op"] == "adaln":
        t, v = TYPES[c["type"]], c["vecs"]
        s["x"] = _activations(g, c["rows"], c["dim"], t)
        s["shift"], s["scale1"] = _normal(g, v, c["dim"], type=t) * 0.1, 1 + _normal(g, v, c["dim"], type=t) * 0.2
        if v == 1:
            s["shift"], s["scale1"] = s["shift"][0], s["scale1"][0]
    elif c["op"] == "gemm":
        s["a"], s["a_scale"] = _matrix(_activations(g, c["m"], c["k"], torch.bfloat16))
        s["w"], s["w_scale"] = _matrix(_normal(g, c["n"], c["k"]) * c["k"] ** -0.5)
        s["bias"] = _normal(g, c["n"]) if c["bias"] else None
        if c["tail"] == "residual":
            s["aux"], s["gate"] = _normal(g, c["m"], c["n"]), _normal(g, c["n"])
    elif c["op"] == "kv_write":
        t, b, cap, layers, heads = TYPES[c["type"]], c["batch"], c["capacity"], c["layers"], c["heads"]
        s["kv"] = _activations(g, b * c["tokens"], layers * 2 * heads * 128, t)
        s["cache"] = torch.randint(0, 120, (b, cap, layers, 2, heads, 128), generator=g, device="cuda", dtype=torch.uint8).view(E4M3)
        s["scale"] = torch.randint(110, 130, (b, layers, 2, heads, cap), generator=g, device="cuda", dtype=torch.uint8).view(E8M0)
        # a single token goes behind each sequence; a prompt fills the cache from its start, up to its own length
        s["start"] = torch.randint(0, cap, (b,), generator=h, dtype=torch.int32).cuda() if c["tokens"] == 1 else None
        s["lens"] = None if c["tokens"] == 1 else _lengths(h, b, c["tokens"]).cuda()
        s["w"] = 1 + _normal(g, layers, heads, 128, type=t) * 0.1 if c["norm"] else None
        s["rope"] = _rope(4 * cap) if c["rope"] else None
    else:
        b, r, n, heads = c["prompts"], c["groups"], c["queries"], c["heads"]
        own_kv = _normal(g, b * r, n, 4 if c["gate"] else 3, heads, 128)  # q, k, v, gate of one projection
        s["q"], s["k"], s["v"] = own_kv[:, :, 0], own_kv[:, :, 1], own_kv[:, :, 2]
        s["gate"] = own_kv[:, :, 3] if c["gate"] else None
        s["cached"] = []
        for i, cap in enumerate((c["text"], c["speaker"])):
            if not cap:
                continue
            data, e = _quantized(_normal(g, b, cap, 2, heads, 128).float())
            lens = _lengths(h, b, cap)
            # guided rows: [both | without text | without speaker]
            rows = lens if r == 1 else torch.cat([torch.zeros_like(lens) if k == i + 1 else lens for k in range(3)])
            s["cached"].append((data.to(E4M3), e[..., 0].permute(0, 2, 3, 1).contiguous().view(E8M0), rows.cuda()))
    return s


# ------------------------------------------------------------------------------------------------ the plain forms

def _quantized(x):
    """e4m3 values (in fp32) and e8m0 bytes [..., blocks] of fp32 x [..., cols]."""
    cols = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    bits = b.abs().amax(-1).contiguous().view(torch.int32)
    # amax = f * 2^(e - 127) with 1 <= f < 2: 448 = 1.75 * 2^8, so the scale's exponent is e - 8, one more where f > 1.75
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=0)
    q = (b * torch.exp2(127.0 - e)[..., None]).to(E4M3)
    return q.float().flatten(-2)[..., :cols], e.to(torch.uint8)


def _words(e):
    """e8m0 bytes [rows, blocks] as [ceil(blocks / 4), rows, 4]."""
    e = torch.nn.functional.pad(e, (0, -e.shape[1] % 4))
    return e.unflatten(1, (-1, 4)).transpose(0, 1).contiguous().view(E8M0)


def _values(q, words, type=torch.float32):
    """What a matrix in the 8-bit format stands for."""
    f = words.to(type).transpose(0, 1).flatten(1).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    return q.to(type) * f


def _normed(x, weight, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _per_row(v, rows):
    return v if v.dim() == 1 else v.repeat_interleave(rows // v.shape[0], 0)


def _gated(a):
    """SwiGLU of columns in blocks of 16: 16 of the one factor, 16 of the other."""
    a = a.unflatten(1, (-1, 2, 16))
    return (a[:, :, 0] * torch.sigmoid(a[:, :, 0]) * a[:, :, 1]).flatten(1)


def _product(s, type):
    y = _values(s["a"], s["a_scale"], type) @ _values(s["w"], s["w_scale"], type).t()
    if s["bias"] is not None:
        y = y + s["bias"].to(type)
    tail = s["case"]["tail"]
    if tail == "residual":
        return s["aux"].to(type) + s["gate"].to(type) * y
    return y if tail == "store" else _gated(y)


def _rotated(k, rope, heads, positions):
    """Interleaved pairs of the first `heads` heads of k [..., layers, heads, 128], a position for each of the leading axes."""
    cs = rope[positions].to(k.dtype)[..., None, None, :, :]
    a, b = k[..., :heads, 0::2], k[..., :heads, 1::2]
    turned = torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)
    return torch.cat([turned, k[..., heads:, :]], -2)


def _keys_values(s, type):
    """[batch, tokens, layers, 2, heads, 128] as the cache is to hold them, and the slot of each token."""
    c = s["case"]
    kv = s["kv"].to(type).reshape(c["batch"], c["tokens"], c["layers"], 2, c["heads"], 128)
    k, v = kv[:, :, :, 0], kv[:, :, :, 1]
    at = torch.arange(c["tokens"], device="cuda").expand(c["batch"], -1)
    if s["start"] is not None:
        at = at + s["start"][:, None]
    if s["w"] is not None:
        k = _normed(k, s["w"].to(type), EPS)
    if s["rope"] is not None:
        k = _rotated(k, s["rope"], c["rope"], at * 4)
    return torch.stack([k, v], 3), at


def _attention(s, type):
    """Softmax over what each row sees of its own sequence and of the caches; a row that sees nothing is zero."""
    c = s["case"]
    q = s["q"].to(type)
    rows, n = q.shape[:2]
    ks, vs, seen = [], [], []
    if c["self"]:
        ks.append(s["k"].to(type)), vs.append(s["v"].to(type))
        seen.append(torch.ones((rows, n), dtype=torch.bool, device="cuda"))
    for data, scale, lens in s["cached"]:
        kv = data.to(type) * scale.to(type).permute(0, 3, 1, 2)[..., None]
        kv = kv.repeat(c["groups"], 1, 1, 1, 1)
        ks.append(kv[:, :, 0]), vs.append(kv[:, :, 1])
        seen.append(torch.arange(kv.shape[1], device="cuda") < lens[:, None])
    seen = torch.cat(seen, 1)[:, None, None]
    scores = q.transpose(1, 2) @ torch.cat(ks, 1).permute(0, 2, 3, 1).contiguous() * 128 ** -0.5
    scores = scores.masked_fill_(~seen, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    o = scores @ torch.cat(vs, 1).transpose(1, 2).contiguous() / scores.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.transpose(1, 2)
    return o if s["gate"] is None else o * torch.sigmoid(s["gate"].to(type))


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        q, e = _quantized(s["x"].float())
        return q.to(E4M3), _words(e)
    if c["op"] == "adaln":
        y = _normed(s["x"].float(), _per_row(s["scale1"].float(), c["rows"]), EPS) + _per_row(s["shift"].float(), c["rows"])
        q, e = _quantized(y)
        return q.to(E4M3), _words(e)
    if c["op"] == "gemm":
        y = _product(s, torch.float32)
        if c["tail"] != "swiglu_fp8":
            return y.to(torch.bfloat16)
        q, e = _quantized(y)
        return q.to(E4M3), _words(e)
    if c["op"] == "kv_write":
        kv, at = _keys_values(s, torch.float32)
        q, e = _quantized(kv)
        keep = torch.ones_like(at, dtype=torch.bool) if s["lens"] is None else at < s["lens"][:, None]
        b, t = keep.nonzero(as_tuple=True)
        s["cache"].view(torch.uint8)[b, at[b, t]] = q[b, t].to(E4M3).view(torch.uint8)
        s["scale"].view(torch.uint8)[b, :, :, :, at[b, t]] = e[b, t, ..., 0]
        return s["cache"], s["scale"]
    return _attention(s, torch.float32).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    if not own:
        return _plain(state)
    from echo_tts_amd import _lib, ops
    s, c = state, state["case"]
    if c["op"] == "quantize":
        return ops.quantize_fp8(s["x"])
    if c["op"] == "adaln":
        return ops.adaln_modulate_fp8(s["x"], s["shift"], s["scale1"], EPS)
    if c["op"] == "gemm":
        a = (s["a"], s["a_scale"], s["w"], s["w_scale"])
        if c["tail"] == "store":
            return ops.gemm_fp8(*a, bias=s["bias"])
        if c["tail"] == "residual":
            return ops.gemm_fp8(*a, bias=s["bias"], epilogue=_lib.EPI_RESID, aux=s["aux"], gate=s["gate"])
        return ops.gemm_fp8(*a, epilogue=_lib.EPI_SWIGLU, quantize=c["tail"] == "swiglu_fp8")
    if c["op"] == "kv_write":
        ops.kv_write_fp8(s["kv"], s["cache"], s["scale"], start=s["start"], lens=s["lens"], w=s["w"], eps=EPS, rope=s["rope"],
                         rope_heads=c["rope"], pos_mult=4)
        return s["cache"], s["scale"]
    segments = [ops.Segment(s["k"], s["v"])] if c["self"] else []
    for data, scale, lens in s["cached"]:
        segments.append(ops.Segment(data[:, :, 0], data[:, :, 1], lens=lens, k_scale=scale[:, 0], v_scale=scale[:, 1]))
    return ops.attention(s["q"], segments, gate=s["gate"])


# ------------------------------------------------------------------------------------------------ in 64 bits

def _nearest(y):
    """The e4m3 value nearest to each of y, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _blocks64(y):
    """e4m3 values and scales [..., blocks] of y, both in 64 bits."""
    cols = y.shape[-1]
    b = torch.nn.functional.pad(y, (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    f = torch.exp2(torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -127))))
    f = torch.where(amax > 448 * f, f * 2, torch.where(amax <= 224 * f, f / 2, f)).clamp(min=2.0 ** -127)
    return _nearest(b / f[..., None]).flatten(-2)[..., :cols], f


def _words64(f):
    f = torch.nn.functional.pad(f, (0, -f.shape[1] % 4), value=2.0 ** -127)
    return f.unflatten(1, (-1, 4)).transpose(0, 1).contiguous()


def exact(case, seed):
    s, c = prepare(case, seed), case
    d = torch.float64
    if c["op"] in ("quantize", "adaln"):
        y = s["x"].to(d)
        if c["op"] == "adaln":
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
            y = y.unflatten(0, (c["vecs"], -1)) * s["scale1"].to(d).reshape(c["vecs"], 1, -1) + s["shift"].to(d).reshape(c["vecs"], 1, -1)
            y = y.flatten(0, 1)
        q, f = _blocks64(y)
        return q, _words64(f)
    if c["op"] == "gemm":
        def whole(q, w):
            f = w.to(d).permute(1, 0, 2).reshape(q.shape[0], -1, 1)
            blocks = torch.nn.functional.pad(q.to(d), (0, -q.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
            return (blocks * f[:, :blocks.shape[1]]).flatten(1)
        y = whole(s["a"], s["a_scale"]).mm(whole(s["w"], s["w_scale"]).t())
        if s["bias"] is not None:
            y += s["bias"].to(d)
        if c["tail"] == "store":
            return y
        if c["tail"] == "residual":
            return s["aux"].to(d) + y * s["gate"].to(d)
        y = y.reshape(c["m"], c["n"] // 32, 32)
        y = (y[..., :16] / (1 + torch.exp(-y[..., :16])) * y[..., 16:]).reshape(c["m"], -1)
        if c["tail"] == "swiglu":
            return y
        q, f = _blocks64(y)
        return q, _words64(f)
    if c["op"] == "kv_write":
        cache, scale = s["cache"].to(d), s["scale"].to(d)
        for b in range(c["batch"]):
            n = c["tokens"] if s["lens"] is None else int(s["lens"][b])
            first = 0 if s["start"] is None else int(s["start"][b])
            kv = s["kv"][b * c["tokens"]:b * c["tokens"] + n].to(d).reshape(n, c["layers"], 2, c["heads"], 128).clone()
            k = kv[:, :, 0]
            if s["w"] is not None:
                k = k / (k.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w"].to(d)
            if c["rope"]:
                cs = torch.view_as_complex(s["rope"][4 * first:4 * (first + n):4].to(d).contiguous())[:, None, None]
                z = torch.view_as_complex(k[:, :, :c["rope"]].reshape(n, c["layers"], c["rope"], 64, 2).contiguous())
                k[:, :, :c["rope"]] = torch.view_as_real(z * cs).flatten(-2)
            kv[:, :, 0] = k
            q, f = _blocks64(kv)
            cache[b, first:first + n] = q
            scale[b, :, :, :, first:first + n] = f[..., 0].permute(1, 2, 3, 0)
        return cache, scale
    out = torch.zeros(s["q"].shape, dtype=d, device="cuda")
    for r in range(out.shape[0]):
        ks, vs = ([s["k"][r].to(d)], [s["v"][r].to(d)]) if c["self"] else ([], [])
        for data, scale, lens in s["cached"]:
            b, n = r % c["prompts"], int(lens[r])
            kv = data[b, :n].to(d) * scale[b, :, :, :n].to(d).permute(2, 0, 1)[..., None]
            ks.append(kv[:, 0]), vs.append(kv[:, 1])
        k, v = torch.cat(ks).permute(1, 0, 2), torch.cat(vs).permute(1, 0, 2)
        if k.shape[1]:
            p = torch.softmax(s["q"][r].to(d).permute(1, 0, 2).bmm(k.transpose(1, 2).contiguous()) / math.sqrt(128), -1)
            out[r] = p.bmm(v.contiguous()).permute(1, 0, 2)
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].to(d)))
