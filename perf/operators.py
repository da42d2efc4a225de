"""What the 4-bit KV cache and packed prompts are measured on.

Three families of cases, each an operator of a serving step:

  cache   KvArena.append + KvArena.read_rows: per-head RMSNorm (Qwen3) and
          rotation of new queries and keys, the keys and values quantised to
          4 bits as they are written, and the same rows read back as values.
  decode  KvArena.decode on a 4-bit arena: one new token per sequence is
          normed, rotated, quantised and appended, then attends its cache.
  prompt  Context.attend_packed: causal grouped-query attention of whole
          prompts packed one after another, of different lengths.

Head layouts are the framework's two: Granite (16 query heads, 8 kv heads,
head_dim 64) and Qwen3 (32, 4, 128).

A 4-bit row holds, per kv head and group of 32 dims, an fp16 scale
(max |x| / 7, rounded to fp16) and 32 codes round(x / scale) in -7..7, ties
to even. Rotated keys are rounded to 32 bits before they are quantised, in
the operation order of each model's rotation.
"""
import functools
import math

import torch

own = False

SHAPE = {"granite": (16, 8, 64), "qwen3": (32, 4, 128)}  # query heads, kv heads, head_dim
SOFTMAX_SCALE = {"granite": 1.0 / 64.0, "qwen3": 1.0 / math.sqrt(128.0)}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32
EPS = 1e-6


def listed():
    return [
        # a single chat session's decode step writes its one new token
        {"name": "cache granite 1 token", "kind": "cache", "model": "granite", "dtype": "f32", "sequences": 1,
         "tokens": 1, "start": 511, "page": 0},
        # a serving step: 61 sequences write one token each, far into their contexts
        {"name": "cache qwen3 61 tokens", "kind": "cache", "model": "qwen3", "dtype": "bf16", "sequences": 61,
         "tokens": 61, "start": 30000, "page": 64},
        # the prompts of a batch of short sessions, uneven lengths
        {"name": "cache granite prompts", "kind": "cache", "model": "granite", "dtype": "bf16", "sequences": 9,
         "tokens": 9001, "start": 0, "page": 0},
        # one long document
        {"name": "cache qwen3 document", "kind": "cache", "model": "qwen3", "dtype": "bf16", "sequences": 1,
         "tokens": 32768, "start": 0, "page": 256},
        # one layer of a short session: latency
        {"name": "decode granite short", "kind": "decode", "model": "granite", "dtype": "f32", "out": "f32",
         "sequences": 1, "longest": 512, "layers": 1, "page": 0, "even": True},
        # the layer stack of one full session
        {"name": "decode granite stack", "kind": "decode", "model": "granite", "dtype": "f32", "out": "f32",
         "sequences": 1, "longest": 4064, "layers": 24, "page": 0, "even": True},
        # one layer of one long session
        {"name": "decode qwen3 long", "kind": "decode", "model": "qwen3", "dtype": "bf16", "out": "bf16",
         "sequences": 1, "longest": 32768, "layers": 1, "page": 0, "even": True},
        # a serving batch of uneven sessions in a paged arena
        {"name": "decode qwen3 batch", "kind": "decode", "model": "qwen3", "dtype": "bf16", "out": "bf16",
         "sequences": 48, "longest": 8190, "layers": 2, "page": 64, "even": False},
        # a large batch, several layers
        {"name": "decode granite batch", "kind": "decode", "model": "granite", "dtype": "bf16", "out": "bf16",
         "sequences": 128, "longest": 4096, "layers": 4, "page": 0, "even": False},
        # a handful of short prompts, one of them a single token, one empty
        {"name": "prompt granite short", "kind": "prompt", "model": "granite", "dtype": "bf16", "sequences": 7,
         "tokens": 777, "fused": True},
        # a batch of uneven prompts straight out of a joint q/k/v projection
        {"name": "prompt qwen3 batch", "kind": "prompt", "model": "qwen3", "dtype": "f16", "sequences": 11,
         "tokens": 12345, "fused": True},
        # one long prompt
        {"name": "prompt qwen3 long", "kind": "prompt", "model": "qwen3", "dtype": "bf16", "sequences": 1,
         "tokens": 16384, "fused": False},
    ]


def _log_size(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("cache", "decode", "prompt"))
    model = rng.choice(("granite", "qwen3"))
    page = rng.choice((0, 64, 128, 512))
    if kind == "cache":
        start = rng.choice((0, _log_size(rng, 1, 2000 if model == "granite" else 30000)))
        sequences = _log_size(rng, 1, 96)
        tokens = max(sequences, _log_size(rng, 1, min(2048, 4096 - start) if model == "granite" else 8000))
        return {"kind": kind, "model": model, "dtype": rng.choice(("f32", "bf16", "f16")), "sequences": sequences,
                "tokens": tokens, "start": start, "page": page}
    if kind == "decode":
        sequences, layers = _log_size(rng, 1, 96), rng.choice((1, 1, 2, 3))
        longest = _log_size(rng, 1, 4096 if model == "granite" else min(40960, 400000 // (sequences * layers)))
        return {"kind": kind, "model": model, "dtype": rng.choice(("f32", "bf16", "f16")),
                "out": rng.choice(("f32", "bf16", "f16")), "sequences": sequences, "longest": longest,
                "layers": layers, "page": page, "even": rng.random() < 0.3}
    sequences = _log_size(rng, 1, 40)
    return {"kind": kind, "model": model, "dtype": rng.choice(("bf16", "f16")), "sequences": sequences,
            "tokens": max(sequences, _log_size(rng, 20, 12000)), "fused": rng.random() < 0.5}


# ---- sizes of a case ----------------------------------------------------------
def _shares(total, parts, seed):
    """`parts` uneven whole numbers that add up to `total`: with three parts or more one is 0 and one is 1 where
    the total allows it."""
    if parts == 1:
        return [total]
    g = torch.Generator().manual_seed(seed)
    weight = torch.rand(parts, generator=g, dtype=torch.float64) + 0.05
    got = [int(x) for x in torch.floor(weight / weight.sum() * total)]
    if parts >= 3 and total >= 2 * parts:
        got[1], got[parts // 2 + 1] = 0, 1
    got[0] += total - sum(got)
    return got


def _counts(case):
    n = case["sequences"]
    return [1] * n if case["tokens"] == n else _shares(case["tokens"], n, 17 * n + case["tokens"])


def _attended(case):
    """Cached positions of each sequence of a decode case, its new token among them."""
    n, longest = case["sequences"], case["longest"]
    if case["even"]:
        return [longest] * n
    g = torch.Generator().manual_seed(31 * n + longest)
    got = [1 + int(x * (longest - 1)) for x in torch.rand(n, generator=g, dtype=torch.float64)]
    got[-1] = longest
    if n > 2:
        got[1] = 1
    return got


def work(case):
    hq, hkv, d = SHAPE[case["model"]]
    es = 4 if case["dtype"] == "f32" else 2
    row = 2 * hkv * (d // 2 + d // GROUP * 2)  # one position's 4-bit keys and values
    if case["kind"] == "cache":
        t = case["tokens"]
        return {"bytes": t * (hq * d * (es + 2) + 2 * hkv * d * (es + 2) + row + d // 2 * 8),
                "flops": t * (hq + 2 * hkv) * d * 6}
    if case["kind"] == "decode":
        rows, units = sum(_attended(case)) * case["layers"], case["sequences"] * case["layers"]
        eo = 4 if case["out"] == "f32" else 2
        return {"bytes": rows * row + units * (hq * d * (es + eo) + 2 * hkv * d * es), "flops": 4 * rows * hq * d}
    t = case["tokens"]
    return {"bytes": t * (2 * hq + 2 * hkv) * d * 2,
            "flops": sum(2 * hq * d * n * (n + 1) for n in _counts(case))}


# ---- rotation tables ------------------------------------------------------------
def _fma(a, b, c):
    return (a.double() * b.double() + c.double()).float()


@functools.lru_cache(maxsize=None)
def _frequencies(model):
    d = SHAPE[model][2]
    theta = 10000.0 if model == "granite" else 1000000.0
    return torch.tensor([theta ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64).float()


def _bits(*words):
    return torch.tensor(words, dtype=torch.int64).to(torch.int32).view(torch.float32).tolist()


def _table(model, positions, device="cuda"):
    """(cos, sin) [positions][head_dim / 2] in 32 bits, of the angle position * frequency in 32 bits. Granite's are
    qx's pinned polynomials, in their operation order."""
    angle = torch.arange(positions, device=device, dtype=torch.float32)[:, None] * _frequencies(model).to(device)
    if model == "qwen3":
        return angle.double().cos().float(), angle.double().sin().float()
    per_turn, turn_hi, turn_lo, half_pi, pi = _bits(0x3e22f983, 0x40c90fdb, 0xb43bbd2e - (1 << 32), 0x3fc90fdb,
                                                    0x40490fdb)
    sine = _bits(0x2f309231, 0xb2d7322b - (1 << 32), 0x3638ef1d, 0xb9500d01 - (1 << 32), 0x3c088889,
                 0xbe2aaaab - (1 << 32))
    cosine = _bits(0x310f76c7, 0xb493f27e - (1 << 32), 0x37d00d01, 0xbab60b61 - (1 << 32), 0x3d2aaaab,
                   0xbf000000 - (1 << 32))
    const = lambda v: torch.full((), v, dtype=torch.float32, device=device)  # noqa: E731
    turns = torch.trunc(angle * const(per_turn) + 0.5)
    r = _fma(-turns, const(turn_lo), _fma(-turns, const(turn_hi), angle))
    over, under = r > half_pi, r < -half_pi
    r = torch.where(over, const(pi) - r, torch.where(under, const(-pi) - r, r))
    sign = torch.where(over | under, -1.0, 1.0)
    sq = r * r
    s = functools.reduce(lambda acc, c: _fma(acc, sq, const(c)), sine[1:], const(sine[0]).expand_as(sq))
    c = functools.reduce(lambda acc, c: _fma(acc, sq, const(c)), cosine[1:], const(cosine[0]).expand_as(sq))
    return _fma(c, sq, const(1.0)) * sign, _fma(s * sq, r, r)


# ---- inputs -----------------------------------------------------------------------
def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _keys(g, shape, dtype):
    """Keys with a few large channels, as cached keys have."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=g, device="cuda") > 0.97)
    return (x * loud).to(dtype)


_context = None


def _own_context():
    global _context
    from qx_b200 import Context
    if _context is None:
        _context = Context(torch.cuda.current_device())
    _context.set_stream(torch.cuda.current_stream())
    return _context


def _own_arena(case, layers, capacity, rows):
    """A 4-bit arena for sequences of `rows` positions each."""
    import qx_b200 as qx
    model = qx.MODEL_QWEN3 if case["model"] == "qwen3" else qx.MODEL_GRANITE
    page = case["page"]
    pool = sum(-(-n // page) for n in rows) if page else 0
    return qx.KvArena(_own_context(), model, layers, len(rows), capacity, qx.Q4, page_size=page, pool_pages=max(1, pool))


def _code(name):
    import qx_b200 as qx
    return {"f32": qx.F32, "bf16": qx.BF16, "f16": qx.F16}[name]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    hq, hkv, d = SHAPE[case["model"]]
    dt = DTYPE[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "prompt":
        t = case["tokens"]
        s["lengths"] = _counts(case)
        if case["fused"]:
            joint = torch.randn((t, hq + 2 * hkv, d), generator=g, device="cuda")
            joint[:, :hq] *= 1.5
            joint = joint.to(dt)
            s["q"], s["k"], s["v"] = joint[:, :hq], joint[:, hq:hq + hkv], joint[:, hq + hkv:]
        else:
            s["q"], s["k"], s["v"] = _normal(g, (t, hq, d), dt, 1.5), _keys(g, (t, hkv, d), dt), _normal(g, (t, hkv, d), dt)
        if own:
            _own_context()
            s["out"] = torch.zeros((t, hq, d), dtype=dt, device="cuda")
        return s
    s["q_norm"] = s["k_norm"] = None
    if case["model"] == "qwen3":
        s["q_norm"] = 1.0 + 0.3 * torch.rand(d, generator=g, device="cuda")
        s["k_norm"] = 1.0 + 0.3 * torch.rand(d, generator=g, device="cuda")
    if case["kind"] == "cache":
        t, start = case["tokens"], case["start"]
        s["counts"] = _counts(case)
        s["starts"] = [start] * case["sequences"]
        end = start + max(s["counts"])
        s["q"], s["k"], s["v"] = _normal(g, (t, hq, d), dt, 1.5), _keys(g, (t, hkv, d), dt), _normal(g, (t, hkv, d), dt)
        if own:
            s["arena"] = _own_arena(case, 1, end, [start + n for n in s["counts"]])
            for i in range(case["sequences"]):
                s["arena"].set_len(i, start)
            s["rot"] = torch.zeros((t, hq, d), dtype=torch.bfloat16, device="cuda")
            s["keys"] = torch.zeros((t, hkv, d), dtype=torch.bfloat16, device="cuda")
            s["values"] = torch.zeros((t, hkv, d), dtype=torch.bfloat16, device="cuda")
        else:
            s["table"] = _table(case["model"], end)
        return s
    attended, layers = _attended(case), case["layers"]
    n = len(attended)
    s["positions"] = [a - 1 for a in attended]
    s["q"] = _normal(g, (n, layers, hq, d), dt, 1.5)
    s["k"], s["v"] = _keys(g, (n, layers, hkv, d), dt), _normal(g, (n, layers, hkv, d), dt)
    total = sum(s["positions"])
    if own:
        s["arena"] = _own_arena(case, layers, max(attended), attended)
        s["out"] = torch.zeros((n, layers, hq, d), dtype=DTYPE[case["out"]], device="cuda")
        s["keys"] = torch.zeros((n, layers, hkv, d), dtype=torch.bfloat16, device="cuda")
        s["values"] = torch.zeros((n, layers, hkv, d), dtype=torch.bfloat16, device="cuda")
    else:
        s["table"] = _table(case["model"], max(attended))
        longest = max(attended)
        for name in ("key", "value"):
            s[name + "_codes"] = torch.zeros((n, layers, longest, hkv, d // 2), dtype=torch.uint8, device="cuda")
            s[name + "_scales"] = torch.zeros((n, layers, longest, hkv, d // GROUP), dtype=torch.float16, device="cuda")
        at = torch.cat([torch.arange(p) for p in s["positions"]]).cuda()
        which = torch.repeat_interleave(torch.arange(n), torch.tensor(s["positions"])).cuda()
        s["attended"] = torch.tensor(attended, device="cuda")
    # the cached rows before the new token, layer by layer, as an earlier step wrote them
    for layer in range(layers):
        k, v = _keys(g, (total, hkv, d), dt), _normal(g, (total, hkv, d), dt)
        if own:
            for i in range(n):
                s["arena"].set_len(i, 0)
            s["arena"].append(None, k, v, positions=[0] * n, counts=s["positions"], layer_begin=layer, layer_count=1,
                              in_dtype=_code(case["dtype"]), k_norm=s["k_norm"])
        else:
            k = _rotated(case["model"], k, s["k_norm"], at, s["table"])
            for name, x in (("key", k), ("value", v.float())):
                codes, scales = _quantised(x)
                s[name + "_codes"][which, layer, at] = _packed(codes)
                s[name + "_scales"][which, layer, at] = scales
    if own:
        for i, p in enumerate(s["positions"]):
            s["arena"].set_len(i, p)
    return s


# ---- plain forms --------------------------------------------------------------------
def _rotated(model, x, norm, at, table):
    """Rows x [t, heads, head_dim] normed (Qwen3) and rotated to positions `at`, in 32 bits."""
    d = x.shape[-1]
    x = x.float()
    cos, sin = (part[at][:, None, :] for part in table)
    if model == "granite":
        left, right = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([_fma(-right, sin, left * cos), _fma(right, cos, left * sin)], dim=-1)
    mean = x.double().square().sum(-1, keepdim=True) / d
    x = x * (1.0 / torch.sqrt(mean + EPS)).float()
    if norm is not None:
        x = x * norm
    left, right = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([left * cos - right * sin, right * cos + left * sin], dim=-1)


def _quantised(x):
    """Codes -7..7 [..., head_dim] and fp16 scales [..., head_dim / 32] of 32-bit rows."""
    groups = x.unflatten(-1, (-1, GROUP))
    scales = (groups.abs().amax(-1) / torch.full((), 7.0, device=x.device)).half()
    by = scales.float()[..., None]
    codes = torch.where(by > 0, torch.round(groups / by).clamp(-7, 7), torch.zeros_like(groups))
    return codes.flatten(-2).to(torch.int8), scales


def _packed(codes):
    low = (codes + 7).to(torch.uint8)
    return low[..., 0::2] | (low[..., 1::2] << 4)


def _values(codes, scales):
    """The 32-bit values of codes -7..7 and their scales."""
    return (codes.float().unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _unpacked(packed, scales):
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    return _values(codes.to(torch.int8) - 7, scales)


def _ragged(starts, counts, device="cuda"):
    """Position of every packed token."""
    starts, counts = torch.tensor(starts), torch.tensor(counts)
    first = torch.cumsum(counts, 0) - counts
    return (torch.arange(int(counts.sum())) + torch.repeat_interleave(starts - first, counts)).to(device)


def _plain_cache(s):
    model = s["case"]["model"]
    at = _ragged(s["starts"], s["counts"])
    q = _rotated(model, s["q"], s["q_norm"], at, s["table"])
    k = _rotated(model, s["k"], s["k_norm"], at, s["table"])
    keys, values = _values(*_quantised(k)), _values(*_quantised(s["v"].float()))
    return {"q": q.bfloat16(), "keys": keys.bfloat16(), "values": values.bfloat16()}


def _plain_decode(s):
    model = s["case"]["model"]
    hq, hkv, d = SHAPE[model]
    n, layers = s["q"].shape[:2]
    last = s["attended"] - 1
    at = last.repeat_interleave(layers)
    q = _rotated(model, s["q"].flatten(0, 1), s["q_norm"], at, s["table"])
    k = _rotated(model, s["k"].flatten(0, 1), s["k_norm"], at, s["table"])
    each = torch.arange(n, device="cuda")
    for name, x in (("key", k), ("value", s["v"].flatten(0, 1).float())):
        codes, scales = _quantised(x)
        s[name + "_codes"][each, :, last] = _packed(codes).unflatten(0, (n, layers))
        s[name + "_scales"][each, :, last] = scales.unflatten(0, (n, layers))
    keys = _unpacked(s["key_codes"], s["key_scales"])
    q = q.view(n, layers, hkv, hq // hkv, d)
    scores = torch.einsum("nlhgd,nlthd->nlhgt", q, keys) * SOFTMAX_SCALE[model]
    del keys
    outside = torch.arange(scores.shape[-1], device="cuda") >= s["attended"][:, None]
    scores.masked_fill_(outside[:, None, None, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("nlhgt,nlthd->nlhgd", p, _unpacked(s["value_codes"], s["value_scales"])) / total
    last_rows = {name: _unpacked(s[name + "_codes"][each, :, last], s[name + "_scales"][each, :, last])
                 for name in ("key", "value")}
    return {"out": out.reshape(n, layers, hq, d).to(DTYPE[s["case"]["out"]]), "keys": last_rows["key"].bfloat16(),
            "values": last_rows["value"].bfloat16()}


def _plain_prompt(s):
    hq, hkv, d = SHAPE[s["case"]["model"]]
    outs = []
    for q, k, v in zip(*(torch.split(s[name], s["lengths"]) for name in ("q", "k", "v"))):  # prompts differ in length
        length = q.shape[0]
        q = q.float().view(length, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        k, v = k.float().permute(1, 0, 2), v.float().permute(1, 0, 2)
        out = torch.empty((hkv, hq // hkv, length, d), device="cuda")
        hidden = torch.ones((length, length), dtype=torch.bool, device="cuda").triu(1)
        for h in range(hkv):  # one kv head at a time: the scores of all would not fit
            scores = torch.matmul(q[h], k[h].t()) * SOFTMAX_SCALE[s["case"]["model"]]
            scores.masked_fill_(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True)) if length else scores
            out[h] = torch.matmul(p, v[h]) / p.sum(-1, keepdim=True)
        outs.append(out.permute(2, 0, 1, 3).reshape(length, hq, d).to(s["q"].dtype))
    return {"out": torch.cat(outs)}


def run(s):
    case = s["case"]
    if not own:
        return {"cache": _plain_cache, "decode": _plain_decode, "prompt": _plain_prompt}[case["kind"]](s)
    import qx_b200 as qx
    if case["kind"] == "prompt":
        model = qx.MODEL_QWEN3 if case["model"] == "qwen3" else qx.MODEL_GRANITE
        _context.attend_packed(model, s["q"], s["k"], s["v"], s["out"], s["lengths"], dtype=_code(case["dtype"]))
        return {"out": s["out"]}
    if case["kind"] == "cache":
        s["arena"].append(s["q"], s["k"], s["v"], positions=s["starts"], counts=s["counts"], q_rot=s["rot"],
                          in_dtype=_code(case["dtype"]), rot_dtype=qx.BF16, q_norm=s["q_norm"], k_norm=s["k_norm"],
                          flags=qx.DECODE_NO_ADVANCE)
        s["arena"].read_rows(s["keys"], s["values"], begins=s["starts"], counts=s["counts"], out_dtype=qx.BF16)
        return {"q": s["rot"], "keys": s["keys"], "values": s["values"]}
    n = s["k"].shape[0]
    s["arena"].decode(s["q"], s["k"], s["v"], s["out"], s["positions"], q_dtype=_code(case["dtype"]),
                      in_dtype=_code(case["dtype"]), out_dtype=_code(case["out"]), q_norm=s["q_norm"],
                      k_norm=s["k_norm"], flags=qx.DECODE_NO_ADVANCE)
    s["arena"].read_rows(s["keys"], s["values"], begins=s["positions"], counts=[1] * n, out_dtype=qx.BF16)
    return {"out": s["out"], "keys": s["keys"], "values": s["values"]}


# ---- the definition in 64 bits ----------------------------------------------------------
def _exact_rotation(model, x, norm, at):
    x = x.double()
    half = x.shape[-1] // 2
    if model == "qwen3":
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = x if norm is None else x * norm.double()
    angle = (at.float()[:, None] * _frequencies(model).cuda()).double()[:, None, :]
    turned = torch.view_as_complex(torch.stack((x[..., :half], x[..., half:]), -1)) * torch.polar(
        torch.ones_like(angle), angle)
    return torch.cat((turned.real, turned.imag), -1)


def _exact_stored(x):
    """What a 4-bit row holds for x, as values."""
    out = torch.empty_like(x)
    for begin in range(0, x.shape[-1], GROUP):
        part = x[..., begin:begin + GROUP]
        scale = (part.abs().max(-1, keepdim=True).values / 7.0).to(torch.float16).double()
        steps = torch.where(scale == 0, torch.zeros_like(part), (part / scale).round().clamp(-7.0, 7.0))
        out[..., begin:begin + GROUP] = steps * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    model = case["model"]
    hq, hkv, d = SHAPE[model]
    if case["kind"] == "cache":
        at = torch.cat([torch.arange(a, a + c) for a, c in zip(s["starts"], s["counts"])]).cuda()
        return {"q": _exact_rotation(model, s["q"], s["q_norm"], at),
                "keys": _exact_stored(_exact_rotation(model, s["k"], s["k_norm"], at)),
                "values": _exact_stored(s["v"].double())}
    if case["kind"] == "prompt":
        out = torch.empty((case["tokens"], hq, d), dtype=torch.float64, device="cuda")
        begin = 0
        for length in s["lengths"]:
            rows = slice(begin, begin + length)
            for h in range(hq):
                k, v = (s[name][rows, h // (hq // hkv)].double() for name in ("k", "v"))
                for at in range(0, length, 2048):
                    q = s["q"][rows, h][at:at + 2048].double()
                    seen = min(length, at + q.shape[0])
                    logits = q @ k[:seen].T * SOFTMAX_SCALE[model]
                    later = torch.arange(seen, device="cuda") > torch.arange(at, seen, device="cuda")[:, None]
                    out[begin + at:begin + seen, h] = torch.softmax(logits.masked_fill(later, -math.inf), -1) @ v[:seen]
            begin += length
        return {"out": out}
    n, layers = s["q"].shape[:2]
    out = torch.empty((n, layers, hq, d), dtype=torch.float64, device="cuda")
    at = torch.tensor(s["positions"], device="cuda").repeat_interleave(layers)
    q = _exact_rotation(model, s["q"].flatten(0, 1), s["q_norm"], at).view(n, layers, hq, d)
    new_k = _exact_stored(_exact_rotation(model, s["k"].flatten(0, 1), s["k_norm"], at)).view(n, layers, hkv, d)
    new_v = _exact_stored(s["v"].double())
    for i, position in enumerate(s["positions"]):
        for layer in range(layers):
            # the rows before the new token are inputs: what an earlier step stored
            keys, values = (torch.cat((_unpacked(s[name + "_codes"][i, layer, :position],
                                                 s[name + "_scales"][i, layer, :position]).double(), new[i, layer][None]))
                            for name, new in (("key", new_k), ("value", new_v)))
            logits = torch.einsum("hgd,thd->hgt", q[i, layer].view(hkv, hq // hkv, d), keys) * SOFTMAX_SCALE[model]
            out[i, layer] = torch.einsum("hgt,thd->hgd", torch.softmax(logits, -1), values).reshape(hq, d)
    return {"out": out, "keys": new_k, "values": new_v}
